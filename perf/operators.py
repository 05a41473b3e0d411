"""What is measured of the head operators: the 8-bit product with block scales, layer norm, and dropout without a stored mask.

Each case is one call (or one forward and backward) as a training step or a serving loop makes it.  Where ``own`` is
false ``run`` evaluates the defining formulas with elementary torch operations in 32 bits; where it is true it calls
``yolo_from_scratch_amd``.  ``exact`` evaluates the definitions once more in 64 bits.

Definitions
  blocks of 128: s = 2^e with the smallest e >= -127 such that max|x| <= 448 * 2^e over the block (e = 0 for a block of
      zeros); q = x / s rounded to e4m3, to nearest and ties to even.  Activations and gradients have a scale for each
      row and 128 columns, weights for each 128 x 128.
  served product: y = leaky(Q(x) Q(W)^T + b).  Trained: y = Q(x) Q(W)^T + b, dx = Q(dy) Q(W), dW = Q(dy^T) Q(x^T)^T, db =
      sum of dy over the rows.
  layer norm: over the last axis, biased variance.
  dropout: element e of the row-major tensor is kept iff (philox4x32_10(key=seed, counter=e // 4)[e % 4] >> 8) / 2^24
      >= p; kept values are leaky(x) / (1 - p), the others zero.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 128
TOP = 448.0            # largest finite e4m3 value
EPS = 1e-5
SLOPE = 0.1


def listed():
    return [
        # ---- 8-bit product.  One image through the last layer of the head: latency.
        dict(name="fp8 serve last layer, 1 image", op="fp8", train=False, m=1, n=1470, k=4096, bias=True, act=False),
        # one image through the head's first layer: 205 MB of weights for one row
        dict(name="fp8 serve fc, 1 image", op="fp8", train=False, m=1, n=4096, k=50176, bias=True, act=True),
        # a batch of images through it
        dict(name="fp8 serve fc, 64 images", op="fp8", train=False, m=64, n=4096, k=50176, bias=True, act=True),
        # a linear layer over every cell of 64 feature maps of 14 x 14
        dict(name="fp8 serve cells", op="fp8", train=False, m=12544, n=4096, k=4096, bias=True, act=False),
        # a training step of the head's first layer: weights quantised in the step, all three products
        dict(name="fp8 train fc, 64 images", op="fp8", train=True, m=64, n=4096, k=50176, bias=True, act=False),
        # a training step with ragged sizes: rows and outputs that fill no tile
        dict(name="fp8 train ragged", op="fp8", train=True, m=2009, n=1470, k=4096, bias=True, act=False),
        # ---- layer norm.  The head's hidden vector of one image: latency.
        dict(name="norm serve, 1 image", op="norm", train=False, rows=1, cols=4096, dtype="bf16"),
        # the hidden vectors of a training batch
        dict(name="norm train head", op="norm", train=True, rows=64, cols=4096, dtype="bf16"),
        # over the channels of 64 feature maps of 56 x 56, both directions
        dict(name="norm train 56x56x256", op="norm", train=True, rows=200704, cols=256, dtype="bf16"),
        # an odd width in 32 bits: rows that start at every alignment
        dict(name="norm train odd f32", op="norm", train=True, rows=3001, cols=1471, dtype="f32"),
        # ---- dropout.  The hidden vectors of a training batch, with the activation.
        dict(name="dropout train head", op="dropout", rows=64, cols=4096, dtype="bf16", p=0.2, act=True),
        # feature maps, without one
        dict(name="dropout train 56x56x256", op="dropout", rows=200704, cols=256, dtype="bf16", p=0.5, act=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("fp8", "fp8", "norm", "dropout"))
    if op == "fp8":
        train = rng.random() < 0.4
        m = _spread(rng, 1, 4096 if train else 12544)
        n = _spread(rng, 16, 8192)
        # the widest layer is 50176 x 4096; the product over all rows stays under that of the largest listed case
        k = _spread(rng, 64, max(64, min(50176, 205520896 // n, 210453397504 // (m * n * (3 if train else 1)))))
        return dict(op=op, train=train, m=m, n=n, k=k, bias=rng.random() < 0.7, act=not train and rng.random() < 0.5)
    dtype = rng.choice(("bf16", "f16", "f32"))
    cols = _spread(rng, 64, 50176)
    rows = _spread(rng, 1, max(1, min(200704, 102760448 // (cols * BYTES[dtype]))))
    if op == "norm":
        return dict(op=op, train=rng.random() < 0.7, rows=rows, cols=cols, dtype=dtype)
    return dict(op=op, rows=rows, cols=cols, dtype=dtype, p=round(rng.uniform(0.05, 0.9), 3), act=rng.random() < 0.5)


def _generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        # activations as they leave a LeakyReLU, weights as a linear layer's first ones, gradients of a mean loss
        x = torch.nn.functional.leaky_relu(normal(m, k), SLOPE).to(torch.bfloat16)
        w = (torch.rand(n, k, device="cuda", generator=g) * 2 - 1) / math.sqrt(k)
        b = (torch.rand(n, device="cuda", generator=g) * 2 - 1) / math.sqrt(k) if case["bias"] else None
        s = dict(case, x=x, b=b)
        if case["train"]:
            s.update(x=x.requires_grad_(), w=w.requires_grad_(), b=b.requires_grad_() if b is not None else None,
                     dy=(normal(m, n) / m).to(torch.bfloat16))
        else:
            s["wq"], s["we"] = _stored(w)
        return s
    x = normal(case["rows"], case["cols"])
    if case["op"] == "norm":
        x = (x * (1 + torch.rand(case["rows"], 1, device="cuda", generator=g)) + normal(case["rows"], 1)).to(DTYPES[case["dtype"]])
        w = 1 + 0.1 * normal(case["cols"])
        b = 0.1 * normal(case["cols"])
        s = dict(case, x=x, w=w, b=b)
        if case["train"]:
            s.update(x=x.requires_grad_(), w=w.requires_grad_(), b=b.requires_grad_(),
                     dy=normal(case["rows"], case["cols"]).to(x.dtype))
        return s
    return dict(case, x=x.to(DTYPES[case["dtype"]]).requires_grad_(), seed=int(seed) * 0x9E3779B97F4A7C15 % 2 ** 62,
                dy=normal(case["rows"], case["cols"]).to(DTYPES[case["dtype"]]))


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        if s["op"] == "fp8":
            return _plain_train(s) if s["train"] else _plain_serve(s)
        return _plain_norm(s) if s["op"] == "norm" else _plain_dropout(s)


def _run_own(s):
    import yolo_from_scratch_amd as yfs
    if s["op"] == "fp8" and not s["train"]:
        w = yfs.Fp8Tensor(s["wq"], s["we"], s["k"], (128, 128))
        return yfs.fp8_matmul(s["x"], w, bias=s["b"], slope=SLOPE if s["act"] else None)
    if s["op"] == "norm" and not s["train"]:
        return yfs.layer_norm(s["x"], s["w"], s["b"], EPS)
    if s["op"] == "fp8":
        y = yfs.fp8_linear(s["x"], s["w"], s["b"])
        wanted = {"dx": s["x"], "dw": s["w"], "db": s["b"]}
    elif s["op"] == "norm":
        y = yfs.layer_norm(s["x"], s["w"], s["b"], EPS)
        wanted = {"dx": s["x"], "dw": s["w"], "db": s["b"]}
    else:
        y = yfs.dropout(s["x"], s["p"], s["seed"], slope=SLOPE if s["act"] else 1.0)
        wanted = {"dx": s["x"]}
    wanted = {name: t for name, t in wanted.items() if t is not None}
    got = torch.autograd.grad(y, list(wanted.values()), s["dy"])
    return dict(zip(wanted, got), y=y.detach())


def work(case):
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        if not case["train"]:
            nb = -(-n // BLOCK) * -(-k // BLOCK)
            return {"bytes": 2 * m * k + n * k + nb + 2 * m * n + 4 * n * case["bias"], "flops": 2 * m * n * k}
        return {"bytes": 4 * m * k + 8 * n * k + 4 * m * n + 8 * n * case["bias"], "flops": 6 * m * n * k}
    rows, cols, t = case["rows"], case["cols"], BYTES[case["dtype"]]
    if case["op"] == "norm":
        if not case["train"]:
            return {"bytes": 2 * t * rows * cols + 8 * cols, "flops": 8 * rows * cols}
        # the input, y, dy and dx, and the input again for the backward pass
        return {"bytes": 5 * t * rows * cols + 16 * cols, "flops": 22 * rows * cols}
    # x, y, dy, dx, and y again for the activation's sign; twice ten rounds of the generator for four elements
    return {"bytes": (5 if case["act"] else 4) * t * rows * cols, "flops": 32 * rows * cols}


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _pad(x, rows, cols):
    """x with zeros behind it, up to whole blocks."""
    out = x.new_zeros(-(-x.shape[0] // rows) * rows, -(-x.shape[1] // cols) * cols)
    out[: x.shape[0], : x.shape[1]] = x
    return out


def _scale_exponent(amax):
    """The smallest whole e >= -127 with amax <= 448 * 2^e; 0 where amax is 0."""
    mant, expo = torch.frexp(amax)                      # amax = mant * 2^expo, 0.5 <= mant < 1;  448 = 0.875 * 2^9
    e = expo - 9 + (mant > 0.875).to(expo.dtype)
    return torch.where(amax > 0, e.clamp(min=-127), torch.zeros_like(e))


def _power(e):
    """2^e for whole e from -127 to 127, put together from its bits: a computed power can be off in its last place."""
    bits = (e.to(torch.int32).clamp(min=-126) + 127) << 23
    return bits.view(torch.float32) * torch.where(e < -126, 0.5, 1.0)


def _blocks(x, rows, cols):
    """x as blocks of rows x cols: [blocks down, rows, blocks across, cols], and each block's exponent, shaped to go with it."""
    p = _pad(x.float(), rows, cols)
    p = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    return p, _scale_exponent(p.abs().amax(3, keepdim=True).amax(1, keepdim=True))


def _stored(w):
    """A weight in 8 bits, as a server keeps it: e4m3 [n, k up to whole blocks] and the E8M0 bytes of its 128 x 128 blocks."""
    p, e = _blocks(w, BLOCK, BLOCK)
    q = (p * _power(-e)).to(torch.float8_e4m3fn)
    across = p.shape[2]
    q = q.view(torch.uint8).reshape(-1, across * BLOCK)[: w.shape[0]].contiguous().view(torch.float8_e4m3fn)
    return q, (e.reshape(-1, across) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _stored_values(q, e, n, k):
    """The values that stored 8-bit weights stand for."""
    s = _power(e.view(torch.uint8).to(torch.int32) - 127)
    s = s.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)
    return (q.float() * s)[:, :k]


def _rounded(x, rows, cols):
    """The values that x has after it went through blocks of 8-bit numbers."""
    p, e = _blocks(x, rows, cols)
    v = (p * _power(-e)).to(torch.float8_e4m3fn).float() * _power(e)
    return v.reshape(v.shape[0] * rows, -1)[: x.shape[0], : x.shape[1]]


def _leaky(v, act):
    return torch.where(v > 0, v, v * SLOPE) if act else v


def _plain_serve(s):
    v = _rounded(s["x"], 1, BLOCK) @ _stored_values(s["wq"], s["we"], s["n"], s["k"]).t()
    if s["b"] is not None:
        v = v + s["b"]
    return _leaky(v, s["act"]).to(torch.bfloat16)


def _plain_train(s):
    x, w, dy = s["x"], _rounded(s["w"], BLOCK, BLOCK), s["dy"]
    v = _rounded(x, 1, BLOCK) @ w.t()
    if s["b"] is not None:
        v = v + s["b"]
    out = {"y": v.to(torch.bfloat16), "dx": (_rounded(dy, 1, BLOCK) @ w).to(torch.bfloat16),
           "dw": _rounded(dy.t(), 1, BLOCK) @ _rounded(x.t(), 1, BLOCK).t()}
    if s["b"] is not None:
        out["db"] = dy.float().sum(0)
    return out


def _plain_norm(s):
    x = s["x"].float()
    mu = x.mean(1, keepdim=True)
    c = x - mu
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    h = c * r
    y = (h * s["w"] + s["b"]).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    g = dy * s["w"]
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * h).sum(0), "db": dy.sum(0)}


def _philox(key, count):
    """philox4x32_10 of the counters 0 .. count - 1: [count, 4] numbers of 32 bits, held in 64."""
    low = 0xFFFFFFFF
    c0 = torch.arange(count, device="cuda")
    c0, c1 = c0 & low, c0 >> 32
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = key & low, key >> 32
    for _ in range(10):        # the generator's rounds; products wrap at 64 bits, which keeps all the bits that are used
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), 1)


def _plain_dropout(s):
    x, dy = s["x"], s["dy"]
    u = _philox(s["seed"], -(-x.numel() // 4)).reshape(-1)[: x.numel()].view(x.shape)
    keep = (u >> 8).float() * 2.0 ** -24 >= torch.tensor(s["p"], device="cuda", dtype=torch.float32)
    scale = 1 / (1 - s["p"])
    y = torch.where(keep, _leaky(x.float(), s["act"]) * scale, 0.0).to(x.dtype)
    dx = torch.where(keep, dy.float() * scale, 0.0)
    if s["act"]:
        dx = torch.where(y > 0, dx, dx * SLOPE)
    return {"y": y, "dx": dx.to(x.dtype)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _two_to(e):
    """2^e in 64 bits, from a table of the host's."""
    return torch.tensor([2.0 ** k for k in range(-200, 201)], dtype=torch.float64, device="cuda")[e.long() + 200]


def _to_e4m3(v):
    """v rounded to e4m3 by arithmetic: a step is 2^-3 of the binade, 2^-9 below 2^-6."""
    a = v.abs()
    lead = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    lead = lead - (_two_to(lead) > a.clamp(min=2.0 ** -6)).double() + (_two_to(lead + 1) <= a).double()
    step = _two_to(lead - 3)
    return torch.round(v / step) * step


def _through_blocks(x, rows, cols):
    """x in 64 bits after e4m3 blocks; the scale by trying powers of two upwards."""
    r, c = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -c % cols, 0, -r % rows))
    t = x.reshape(x.shape[0] // rows, rows, x.shape[1] // cols, cols)
    top = t.abs().amax((1, 3), keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-45) / TOP)) - 1
    e = e + (TOP * _two_to(e) < top).double()
    e = e + (TOP * _two_to(e) < top).double()
    e = torch.where(top > 0, e.clamp(min=-127), torch.zeros_like(e))
    s = _two_to(e)
    return (_to_e4m3(t / s) * s).reshape(x.shape)[:r, :c]


def _uniform_bits(key, count):
    """The first ``count`` numbers of the generator, on the host and with unsigned numbers."""
    u = np.uint64
    low, half = u(2 ** 32 - 1), u(32)
    ctr = np.arange((count + 3) // 4, dtype=u)
    c = [ctr & low, ctr >> half, np.zeros_like(ctr), np.zeros_like(ctr)]
    keys = [key % 2 ** 32, key // 2 ** 32]
    for r in range(10):
        k = [(keys[0] + r * 0x9E3779B9) % 2 ** 32, (keys[1] + r * 0xBB67AE85) % 2 ** 32]
        p, q = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ u(k[0]), q & low, (p >> half) ^ c[3] ^ u(k[1]), p & low]
    return np.stack(c, 1).reshape(-1)[:count]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "fp8":
        x = s["x"]
        if s["train"]:
            w = _through_blocks(s["w"], 128, 128)
        else:       # from the bytes that are kept: sign, four bits of exponent, three of mantissa
            byte = s["wq"].view(torch.uint8).to(torch.int32)
            expo, mant = (byte >> 3) & 15, (byte & 7).double()
            w = torch.where(expo > 0, (1 + mant / 8) * _two_to(expo - 7), mant * 2.0 ** -9)
            w = torch.where(byte > 127, -w, w)
            row = torch.arange(s["n"], device="cuda") // 128
            col = torch.arange(w.shape[1], device="cuda") // 128
            w = (w * _two_to(s["we"].view(torch.uint8).to(torch.int32) - 127)[row][:, col])[:, : s["k"]]
        y = _through_blocks(x, 1, 128) @ w.t()
        if s["b"] is not None:
            y = y + s["b"].double()
        y = torch.nn.functional.leaky_relu(y, SLOPE) if s["act"] else y
        if not s["train"]:
            return y
        dy = s["dy"].double()
        out = {"y": y, "dx": _through_blocks(dy, 1, 128) @ w,
               "dw": _through_blocks(dy.t(), 1, 128) @ _through_blocks(x.t(), 1, 128).t()}
        if s["b"] is not None:
            out["db"] = dy.sum(0)
        return out
    x = s["x"].double()
    if s["op"] == "norm":
        v, mu = torch.var_mean(x, 1, correction=0, keepdim=True)
        h = (x - mu) * torch.rsqrt(v + EPS)
        w, b = s["w"].double(), s["b"].double()
        y = torch.addcmul(b, h, w)
        if not s["train"]:
            return y
        dy = s["dy"].double()
        g, n = dy * w, x.shape[1]
        dx = (n * g - g.sum(1, keepdim=True) - h * (g * h).sum(1, keepdim=True)) * torch.rsqrt(v + EPS) / n
        return {"y": y, "dx": dx, "dw": torch.einsum("rc,rc->c", dy, h), "db": dy.sum(0)}
    # whole numbers decide what is kept: u >= p  <=>  (u >> 8) >= ceil(p * 2^24) for the float32 p
    p32 = torch.tensor(s["p"], dtype=torch.float32).double().item()
    kept = _uniform_bits(s["seed"], x.numel()) // np.uint64(256) >= np.uint64(math.ceil(p32 * 2 ** 24))
    f = torch.from_numpy(kept).to("cuda").view(x.shape).double() / (1 - s["p"])
    act = s["act"]
    slope = torch.where(x > 0, 1.0, SLOPE if act else 1.0)
    return {"y": x * slope * f, "dx": s["dy"].double() * slope * f}
