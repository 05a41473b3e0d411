"""Layer norm (yolo_from_scratch_amd.layer_norm, HipLayerNorm): the 64-bit oracle against torch and against differences on
the CPU, the kernels against the oracle on the GPU.

Tolerances.  u = finfo(dtype).eps / 2 for the one rounding of an output (plus half the smallest subnormal for fp16).  Inside,
everything is fp32: a sum over a row is a chain of at most 64 terms per thread, a tree over 64 lanes and a chain over 16
waves, so its error is below K = 128 steps of 2^-24 of the sum of magnitudes.  eh below is what that makes of h."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import head_ref as hr

DEV = "cuda:0"
K = 128 * 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2, (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -149)


def _h_error(x, eps):
    """Bound of |h_kernel - h|."""
    _, mu, r, h = hr.layer_norm(x, eps=eps)
    mean_abs = np.abs(x).mean(1, keepdims=True)
    shift = K * mean_abs * r                                  # error of the mean, in units of h
    return shift + (K + shift) * np.abs(h) + K * r * np.abs(x - mu), r, h


def _close(got, ref, tol, what):
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - ref) / tol):.3g} x tolerance"


def _check_forward(y, x, w, b, eps, dtype):
    u, tiny = _half_step(dtype)
    ref = hr.layer_norm(x, w, b, eps)[0]
    eh, _, h = _h_error(x, eps)
    aw = 1.0 if w is None else np.abs(w)
    ab = 0.0 if b is None else np.abs(b)
    inner = aw * eh + 2 * 2.0 ** -24 * (aw * np.abs(h) + ab)
    _close(y, ref, u * (np.abs(ref) + inner) + inner + tiny, "y")


def _check_backward(dx, dw, db, dy, x, w, eps, dtype):
    u, tiny = _half_step(dtype)
    rx, rw, rb = hr.layer_norm_bwd(dy, x, w, eps)
    eh, r, h = _h_error(x, eps)
    ag = np.abs(dy) * (1.0 if w is None else np.abs(w))
    ah = np.abs(h)
    mgh, meh = (ag * ah).mean(1, keepdims=True), (ag * eh).mean(1, keepdims=True)
    inner = r * (2 * K * (ag + ag.mean(1, keepdims=True) + ah * mgh) + eh * (mgh + meh) + ah * meh)
    # r itself: relative error below that of h's scale, already in eh at |h| = 1
    inner = inner + K * 4 * r * (ag + ag.mean(1, keepdims=True) + ah * mgh)
    if dx is not None:
        _close(dx, rx, u * (np.abs(rx) + inner) + inner + tiny, "dx")
    chain = (len(x) + 256) * 2.0 ** -24                        # a column's sum: at most one addition per row, then the joins
    if dw is not None:
        _close(dw, rw, chain * (np.abs(dy) * ah).sum(0) + 2 * (np.abs(dy) * eh).sum(0) + 1e-30, "dw")
    if db is not None:
        _close(db, rb, chain * np.abs(dy).sum(0) + 1e-30, "db")


def _inputs(rows, cols, dtype, seed=0, device=DEV):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 7919 + cols)
    x = (torch.randn(rows, cols, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + torch.randn(rows, 1, generator=g)).to(dtype)
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    b = 0.1 * torch.randn(cols, generator=g)
    dy = torch.randn(rows, cols, generator=g).to(dtype)
    return [t.to(device) for t in (x, w, b, dy)]


def _np(t):
    return t.detach().double().cpu().numpy()


# ---- CPU: oracle and refusals ----------------------------------------------------------------------------------------
def test_oracle_against_torch_and_differences():
    rng = np.random.default_rng(0)
    x, w, b, dy = rng.standard_normal((5, 37)), rng.standard_normal(37), rng.standard_normal(37), rng.standard_normal((5, 37))
    xt, wt, bt = [torch.from_numpy(v).requires_grad_() for v in (x, w, b)]
    yt = torch.nn.functional.layer_norm(xt, (37,), wt, bt, 1e-5)
    yt.backward(torch.from_numpy(dy))
    np.testing.assert_allclose(hr.layer_norm(x, w, b)[0], yt.detach().numpy(), rtol=1e-12, atol=1e-12)
    for mine, theirs in zip(hr.layer_norm_bwd(dy, x, w), (xt.grad, wt.grad, bt.grad)):
        np.testing.assert_allclose(mine, theirs.numpy(), rtol=1e-11, atol=1e-12)
    v, step = rng.standard_normal(x.shape), 1e-6
    diff = (dy * (hr.layer_norm(x + step * v, w, b)[0] - hr.layer_norm(x - step * v, w, b)[0])).sum() / (2 * step)
    np.testing.assert_allclose((hr.layer_norm_bwd(dy, x, w)[0] * v).sum(), diff, rtol=1e-7)


def test_refusals():
    import yolo_from_scratch_amd as y
    x = torch.zeros(4, 8)
    for call in (lambda: y.layer_norm(x), lambda: y.layer_norm(x.int()), lambda: y.layer_norm(x.double()),
                 lambda: y.layer_norm(x, torch.ones(7)), lambda: y.layer_norm(x, None, torch.ones(8, 1)),
                 lambda: y.layer_norm(x, torch.ones(8).long()), lambda: y.layer_norm(x, eps=-1.0),
                 lambda: y.layer_norm(x, eps=float("nan")), lambda: y.layer_norm(torch.zeros(())),
                 lambda: y.layer_norm(torch.zeros(4, 0)), lambda: y.HipLayerNorm(8, channels_first=True)(x)):
        with pytest.raises(y.YfsError):
            call()
    lib, one = y.lib(), 4096
    assert lib.yfs_layer_norm_fwd(one, 8, None, None, None, None, None, 4, 8, 1e-5, 0, None) == -1
    assert lib.yfs_layer_norm_fwd(one, 8, None, None, one, None, None, 0, 8, 1e-5, 0, None) == -1
    assert lib.yfs_layer_norm_fwd(one, 8, None, None, one, None, None, 4, 1 << 30, 1e-5, 0, None) == -1
    assert lib.yfs_layer_norm_fwd(one, 8, None, None, one, None, None, 4, 8, -1.0, 0, None) == -1
    assert lib.yfs_layer_norm_fwd(one, 8, None, None, one, None, None, 4, 8, 1e-5, 3, None) == -2
    need = lib.yfs_layer_norm_bwd_workspace_bytes(100000, 64, 1)
    assert need > 0 and lib.yfs_layer_norm_bwd_workspace_bytes(0, 64, 1) == 0
    assert lib.yfs_layer_norm_bwd(one, 64, one, 64, None, one, one, one, one, one, 100000, 64, 1, one, need - 1, None) == -3
    assert lib.yfs_layer_norm_bwd(one, 64, one, 64, None, None, one, one, one, one, 4, 64, 1, None, 0, None) == -1


# ---- GPU -------------------------------------------------------------------------------------------------------------
COLS = [1, 2, 3, 7, 8, 9, 31, 64, 65, 129, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 1470, 2048, 2049, 4096, 4097, 8192,
        16385, 32768, 32771, 50176]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_forward_and_backward(cols, dtype):
    import yolo_from_scratch_amd as yfs
    t = DTYPES[dtype]
    for rows in (1, 5) if cols > 9000 else (1, 67, 301):
        x, w, b, dy = _inputs(rows, cols, t)
        for v in (x, w, b):
            v.requires_grad_()
        y = yfs.layer_norm(x, w, b, 1e-5)
        assert y.dtype == t and y.shape == x.shape and y.is_contiguous()
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert dx.dtype == t and dw.dtype == db.dtype == torch.float32
        _check_forward(_np(y), _np(x), _np(w), _np(b), 1e-5, t)
        _check_backward(_np(dx), _np(dw), _np(db), _np(dy), _np(x), _np(w), 1e-5, t)
        with torch.no_grad():
            assert torch.equal(yfs.layer_norm(x, w, b, 1e-5), y)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(12544, 192), (4099, 1024), (20001, 33)])
def test_many_rows(rows, cols):
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(rows, cols, torch.bfloat16)
    for v in (x, w, b):
        v.requires_grad_()
    y = yfs.layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    _check_forward(_np(y), _np(x), _np(w), _np(b), 1e-5, x.dtype)
    _check_backward(*[_np(v) for v in got], _np(dy), _np(x), _np(w), 1e-5, x.dtype)
    again = torch.autograd.grad(yfs.layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(got, again))            # fixed order of every sum


@pytest.mark.gpu
def test_without_weight_or_bias_and_partial_gradients():
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(37, 300, torch.float32)
    xn, wn, dyn = _np(x), _np(w), _np(dy)
    _check_forward(_np(yfs.layer_norm(x)), xn, None, None, 1e-5, x.dtype)
    _check_forward(_np(yfs.layer_norm(x, None, b, 1e-3)), xn, None, _np(b), 1e-3, x.dtype)
    xg = x.clone().requires_grad_()
    _check_backward(_np(torch.autograd.grad(yfs.layer_norm(xg), xg, dy)[0]), None, None, dyn, xn, None, 1e-5, x.dtype)
    for need in ("w", "b"):                                              # x needs no gradient
        wg, bg = w.clone().requires_grad_(need == "w"), b.clone().requires_grad_(need == "b")
        got, = torch.autograd.grad(yfs.layer_norm(x, wg, bg), wg if need == "w" else bg, dy)
        _check_backward(None, _np(got) if need == "w" else None, _np(got) if need == "b" else None, dyn, xn, wn, 1e-5, x.dtype)
    wh = w.bfloat16().requires_grad_()                                   # a weight of another type keeps it in its gradient
    got, = torch.autograd.grad(yfs.layer_norm(x, wh), wh, dy)
    assert got.dtype == torch.bfloat16
    ref = hr.layer_norm_bwd(dyn, xn, _np(wh))[1]
    np.testing.assert_allclose(_np(got), ref, rtol=2.0 ** -8 + 1e-4, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_offsets_and_shapes(dtype):
    """Rows inside a wider tensor (also at odd offsets), one row expanded, transposed, 1-d, 4-d and channels-last."""
    import yolo_from_scratch_amd as yfs
    t = DTYPES[dtype]
    wide = torch.randn(40, 700, device=DEV).to(t)
    w, b = torch.randn(331, device=DEV), torch.randn(331, device=DEV)
    narrow = torch.randn(331, 40, device=DEV).to(t)
    views = [wide[:, 3:334], wide[::2, 8:339], wide[5:6, :331].expand(7, 331), narrow.t(), wide[3, 1:332],
             wide[:, :662].reshape(4, 10, 2, 331), wide.flatten()[1:1 + 331 * 9].view(9, 331)]
    for x in views:
        dy = torch.randn(x.shape, device=DEV).to(t)
        xg = x.detach().requires_grad_()
        y = yfs.layer_norm(xg, w, b)
        dx, = torch.autograd.grad(y, xg, dy)
        assert y.shape == x.shape and dx.shape == x.shape
        flat = lambda v: _np(v).reshape(-1, 331)   # noqa: E731
        _check_forward(flat(y), flat(x), _np(w), _np(b), 1e-5, t)
        _check_backward(flat(dx), None, None, flat(dy), flat(x), _np(w), 1e-5, t)
    # a gradient with a stride of its own, and an expanded one
    x = torch.randn(20, 331, device=DEV).to(t).requires_grad_()
    y = yfs.layer_norm(x, w, b)
    for dy in (wide[:20, 5:336], wide[:1, :331].expand(20, 331)):
        dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
        _check_backward(_np(dx), None, None, _np(dy), _np(x), _np(w), 1e-5, t)
    m = yfs.HipLayerNorm(48, channels_first=True).to(DEV)
    fmap = torch.randn(2, 48, 5, 7, device=DEV).to(t).contiguous(memory_format=torch.channels_last)
    out = m(fmap)
    assert out.shape == fmap.shape and out.is_contiguous(memory_format=torch.channels_last)
    rows = lambda v: _np(v.permute(0, 2, 3, 1)).reshape(-1, 48)   # noqa: E731
    _check_forward(rows(out), rows(fmap), None, None, 1e-5, t)
    assert torch.equal(m(fmap.contiguous()), out)


@pytest.mark.gpu
def test_special_rows():
    """NaN and infinity stay in their rows; constant rows and rows of very large values; no rows at all."""
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(9, 130, torch.float32)
    clean = yfs.layer_norm(x, w, b)
    dirty = x.clone()
    dirty[2, 5], dirty[4, 129], dirty[6, 0] = float("nan"), float("inf"), -float("inf")
    out = yfs.layer_norm(dirty, w, b)
    for row in range(9):
        if row in (2, 4, 6):
            assert out[row].isnan().all()
        else:
            assert torch.equal(out[row], clean[row])
    const = torch.full((3, 130), 7.25, device=DEV)
    _check_forward(_np(yfs.layer_norm(const, w, b)), _np(const), _np(w), _np(b), 1e-5, const.dtype)
    big = x * 1e15
    _check_forward(_np(yfs.layer_norm(big, w, b)), _np(big), _np(w), _np(b), 1e-5, big.dtype)
    e = torch.empty(0, 130, device=DEV, requires_grad=True)
    wg = w.clone().requires_grad_()
    y = yfs.layer_norm(e, wg, b)
    assert y.shape == (0, 130)
    ge, gw = torch.autograd.grad(y.sum(), (e, wg))
    assert ge.shape == (0, 130) and (gw == 0).all()


@pytest.mark.gpu
def test_nothing_is_written_behind_the_rows():
    from yolo_from_scratch_amd import _lib as L
    rows, cols, pad = 13, 77, 64
    x, w, b, dy = _inputs(rows, cols, torch.bfloat16)
    n = rows * cols
    y = torch.full((n + pad,), 3.0, device=DEV, dtype=torch.bfloat16)
    dx, stats, dw, db = y.clone(), torch.full((2, rows + pad), 3.0, device=DEV), torch.full((cols + pad,), 3.0, device=DEV), torch.full((cols + pad,), 3.0, device=DEV)
    lib, s = L.lib(), torch.cuda.current_stream().cuda_stream
    L.check(lib.yfs_layer_norm_fwd(x.data_ptr(), cols, w.data_ptr(), b.data_ptr(), y.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(),
                                   rows, cols, 1e-5, 1, s), "fwd")
    assert lib.yfs_layer_norm_bwd_workspace_bytes(rows, cols, 1) == 0
    L.check(lib.yfs_layer_norm_bwd(dy.data_ptr(), cols, x.data_ptr(), cols, w.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(),
                                   dx.data_ptr(), dw.data_ptr(), db.data_ptr(), rows, cols, 1, None, 0, s), "bwd")
    assert (y[n:] == 3).all() and (dx[n:] == 3).all() and (stats[:, rows:] == 3).all() and (dw[cols:] == 3).all() and (db[cols:] == 3).all()
    _check_forward(_np(y[:n]).reshape(rows, cols), _np(x), _np(w), _np(b), 1e-5, x.dtype)
    _check_backward(_np(dx[:n]).reshape(rows, cols), _np(dw[:cols]), _np(db[:cols]), _np(dy), _np(x), _np(w), 1e-5, x.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(9, 33), (5, 1030), (40, 2501), (3, 9001)])
def test_library_on_rows_that_share_no_alignment(rows, cols, dtype):
    """Odd widths through the library itself: rows at a stride of their own and a start at an odd element, forward and backward,
    with guards behind every output."""
    from yolo_from_scratch_amd import _lib as L
    t = DTYPES[dtype]
    x0, w, b, dy0 = _inputs(rows, cols, t)
    big = torch.full((2, rows * (cols + 5) + 8), 2.0, device=DEV).to(t)
    x, dy = [v[1:1 + rows * (cols + 5)].view(rows, cols + 5)[:, :cols] for v in big]
    x.copy_(x0), dy.copy_(dy0)
    y = torch.full((2, rows * cols + 64), 3.0, device=DEV).to(t)
    stats, sums = torch.full((2, rows), 3.0, device=DEV), torch.full((2, cols + 8), 3.0, device=DEV)
    lib, s, code = L.lib(), torch.cuda.current_stream().cuda_stream, L.DTYPES[t]
    L.check(lib.yfs_layer_norm_fwd(x.data_ptr(), cols + 5, w.data_ptr(), b.data_ptr(), y[0].data_ptr(), stats[0].data_ptr(),
                                   stats[1].data_ptr(), rows, cols, 1e-5, code, s), "fwd")
    need = lib.yfs_layer_norm_bwd_workspace_bytes(rows, cols, code)
    ws = torch.full((need + 64,), 7, device=DEV, dtype=torch.uint8)
    dx = y[1, 1:]                                       # an odd start
    L.check(lib.yfs_layer_norm_bwd(dy.data_ptr(), cols + 5, x.data_ptr(), cols + 5, w.data_ptr(), stats[0].data_ptr(),
                                   stats[1].data_ptr(), dx.data_ptr(), sums[0].data_ptr(), sums[1].data_ptr(), rows, cols, code,
                                   ws.data_ptr(), need, s), "bwd")
    n = rows * cols
    assert (y[0, n:] == 3).all() and (dx[n:] == 3).all() and (y[1, :1] == 3).all() and (sums[:, cols:] == 3).all() and (ws[need:] == 7).all()
    _check_forward(_np(y[0, :n]).reshape(rows, cols), _np(x0), _np(w), _np(b), 1e-5, t)
    _check_backward(_np(dx[:n]).reshape(rows, cols), _np(sums[0, :cols]), _np(sums[1, :cols]), _np(dy0), _np(x0), _np(w), 1e-5, t)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", [(9001, 257, "bf16"), (5003, 1470, "f16"), (4100, 3001, "bf16"), (3000, 1471, "f32"),
                                             (20003, 9, "bf16"), (2500, 8193, "bf16"), (1500, 4096, "f16"), (1200, 1536, "bf16"),
                                             (9000, 96, "f32"), (1100, 8192, "f32")])
def test_column_sums_of_many_rows(rows, cols, dtype):
    """Column sums in the pass of dx, with a wave and with a workgroup per row, over rows that begin at every place of an aligned
    16 bytes and over whole ones."""
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(rows, cols, DTYPES[dtype])
    for v in (x, w, b):
        v.requires_grad_()
    y = yfs.layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    _check_forward(_np(y), _np(x), _np(w), _np(b), 1e-5, x.dtype)
    _check_backward(*[_np(v) for v in got], _np(dy), _np(x), _np(w), 1e-5, x.dtype)


@pytest.mark.gpu
def test_gradient_against_differences():
    """<dx, v> against (f(x + sv) - f(x - sv)) / 2s in fp32.  With s = 2^-6 and |v| = 1 a component's rounding enters as
    2^-24 |y| / s = 2^-18 |y dy| (random signs over 4000 terms), the third derivative as s^2 / 6 of order one: 1e-3 of the
    norms covers both."""
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(8, 500, torch.float32)
    x.requires_grad_()
    dx, = torch.autograd.grad(yfs.layer_norm(x, w, b), x, dy)
    v = torch.randn_like(x)
    v = v / v.norm()
    s = 2.0 ** -6
    f = lambda z: (yfs.layer_norm(z, w, b).double() * dy.double()).sum()   # noqa: E731
    with torch.no_grad():
        diff = (f(x + s * v) - f(x - s * v)) / (2 * s)
    assert abs(float((dx.double() * v.double()).sum() - diff)) < 1e-3 * float(dx.norm())


@pytest.mark.gpu
def test_other_stream_and_captured_graph():
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(70000, 64, torch.bfloat16)          # needs a workspace
    for v in (x, w, b):
        v.requires_grad_()

    def step():
        y = yfs.layer_norm(x, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, other))
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.roll(x, 1, 0))
            dy.copy_(dy.flip(0))
        want = step()
        for t in out:
            t.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), k


@pytest.mark.gpu
def test_module_matches_torch_names_and_trains():
    import yolo_from_scratch_amd as yfs
    m, ref = yfs.HipLayerNorm(96).to(DEV), torch.nn.LayerNorm(96)
    assert list(m.state_dict()) == list(ref.state_dict())
    assert list(yfs.HipLayerNorm(96, bias=False).state_dict()) == ["weight"]
    x = torch.randn(12, 96, device=DEV, requires_grad=True)
    m(x).square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in (x, m.weight, m.bias))


def test_library_is_loaded_by_name():
    import yolo_from_scratch_amd as y
    assert hasattr(ctypes.CDLL(y.LIB_PATH), "yfs_layer_norm_bwd")


@pytest.mark.gpu
def test_second_derivative_is_refused():
    import yolo_from_scratch_amd as yfs
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    for f in (lambda: yfs.layer_norm(x), lambda: yfs.dropout(x, 0.5, 1), lambda: yfs.fp8_linear(x, torch.ones(8, 32, device=DEV))):
        with pytest.raises(RuntimeError):
            g, = torch.autograd.grad(f().sum(), x, create_graph=True)
            g.sum().backward()


def test_width_limit():
    import yolo_from_scratch_amd as y
    lib, p, n = y.lib(), 4096, 1 << 28
    assert lib.yfs_layer_norm_fwd(p, n, None, None, p, None, None, 1, n, 1e-5, 0, None) == -1
    assert lib.yfs_layer_norm_bwd(p, n, p, n, None, p, p, p, p, p, 1, n, 0, p, 1 << 40, None) == -1
    assert lib.yfs_layer_norm_bwd_workspace_bytes(1, n, 0) == 0


@pytest.mark.gpu
def test_longest_row():
    """x = +1, -1, ...: mean 2^-28, variance 1; dy = +1, +1, -1, -1, ... has no part along 1 or h.  The sums are exact up to 2^24
    and off by 20 steps of 2^-24 at most behind it, so that y = x and dx = dy after the rounding to bf16."""
    import yolo_from_scratch_amd as yfs
    n = (1 << 28) - 5
    c = torch.arange(n, device=DEV, dtype=torch.int32)
    x = (1 - 2 * (c % 2)).bfloat16()[None].requires_grad_()
    dy = (1 - 2 * (c % 4 // 2)).bfloat16()[None]
    del c
    w, b = torch.ones(n, device=DEV, requires_grad=True), torch.zeros(n, device=DEV, requires_grad=True)
    y = yfs.layer_norm(x, w, b, eps=0.0)
    assert torch.equal(y, x)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(dx, dy) and torch.equal(db, dy[0].float())
    assert float((dw - dy[0].float() * x[0].detach().float()).abs().max()) <= 32 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(5, 8200), (3, 16384), (4, 16392), (3, 20001), (2, 32761), (2, 36693), (2, 50177), (2, 65536), (2, 65543), (1030, 8200),
                                       (1025, 12001), (1100, 16384)])
def test_rows_kept_in_their_own_type(rows, cols, dtype):
    """Widths on both sides of each form of the long rows' kernels, whole vectors and not, with and without sums in the pass of dx."""
    import yolo_from_scratch_amd as yfs
    x, w, b, dy = _inputs(rows, cols, DTYPES[dtype])
    for v in (x, w, b):
        v.requires_grad_()
    y = yfs.layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    if rows > 1000:     # the sums in 64 bits of the whole columns, the rest of a few rows
        xs, wd, dd = x.detach().double(), w.detach().double(), dy.double()
        h = (xs - xs.mean(1, keepdim=True)) / torch.sqrt(xs.var(1, unbiased=False, keepdim=True) + 1e-5)
        tol = (len(xs) + 256) * 2.0 ** -24 * (dd * h).abs().sum(0) + 2 * 8 * K * dd.abs().sum(0)
        assert bool(((got[1].double() - (dd * h).sum(0)).abs() <= tol).all())
        assert bool(((got[2].double() - dd.sum(0)).abs() <= (len(xs) + 256) * 2.0 ** -24 * dd.abs().sum(0)).all())
        pick = [0, 1, rows // 2, rows - 1]
        _check_forward(_np(y[pick]), _np(x[pick]), _np(w), _np(b), 1e-5, x.dtype)
        _check_backward(_np(got[0][pick]), None, None, _np(dy[pick]), _np(x[pick]), _np(w), 1e-5, x.dtype)
        return
    _check_forward(_np(y), _np(x), _np(w), _np(b), 1e-5, x.dtype)
    _check_backward(*[_np(v) for v in got], _np(dy), _np(x), _np(w), 1e-5, x.dtype)
    only = torch.autograd.grad(yfs.layer_norm(x, w.detach(), b.detach()), x, dy)[0]
    assert torch.equal(only, got[0])
