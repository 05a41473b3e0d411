"""The 8-bit product with block scales (yolo_from_scratch_amd.fp8_ops) against the 64-bit oracle.

Quantisers: bytes and scales are compared exactly (powers of two make x / s exact, so one rounding decides).
Products, on the oracle's own quantised operands a, b.  fp32 outputs: the matrix instruction sums 32 products in an order of its
own, K / 32 such sums follow one another and up to 64 parts are joined, so (96 + K / 32) 2^-24 sum|a b|.  16-bit outputs: the
8-bit instruction aligns the 128 products of a block to the largest and keeps 16 bits, so 128 * 2^-16 max|a b| for a block, then
half a step of the output's type."""
import numpy as np
import pytest
import torch

from oracle import head_ref as hr

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _np(t):
    return t.detach().double().cpu().numpy()


def _tolerance(a, b, ref, dtype, extra=0.0):
    """|got - ref| allowed for ref = a b^T + extra rounded to dtype."""
    k = a.shape[1]
    mag = np.abs(a) @ np.abs(b).T
    inner = (96 + k / 32) * 2.0 ** -24 * mag + 2.0 ** -23 * np.abs(extra)
    if dtype != torch.float32:
        for k0 in range(0, k, 128):
            top = np.abs(a[:, None, k0:k0 + 128]) * np.abs(b[None, :, k0:k0 + 128])
            inner = inner + 2.0 ** -9 * top.max(2)
    u = torch.finfo(dtype).eps / 2
    return u * (np.abs(ref) + inner) + inner + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


def _close(got, ref, tol, what):
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - ref) / tol):.3g} x tolerance"


def _matrix(rows, cols, seed, dtype=torch.float32, device=DEV):
    """Values whose size differs from block to block and row to row."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    t = t * torch.exp2(torch.randint(-3, 4, (1, (cols + 127) // 128), generator=g).float()).repeat_interleave(128, 1)[:, :cols]
    return t.to(dtype).to(device)


# ---- CPU -------------------------------------------------------------------------------------------------------------
def test_oracle_rounding_against_torch():
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    v = torch.cat([v[v.abs() <= 448], torch.randn(20000) * torch.exp2(torch.randint(-12, 9, (20000,)).float())])
    v = v[v.abs() <= 448]
    assert np.array_equal(hr.to_e4m3(v.numpy()), v.to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(hr.to_e4m3([480.0, np.inf, -np.inf, np.nan])).all()


def test_oracle_scales():
    amax = np.array([0.0, 448.0, np.nextafter(448.0, 500), 449.0, 1.0, 0.875, 0.8750001, 2.0 ** -133, 3e38])
    e = hr.scale_exponent(amax)
    assert list(e[:3]) == [0, 0, 1]
    for a, k in zip(amax[1:], e[1:]):
        assert a <= 448 * 2.0 ** k and (k == -127 or a > 448 * 2.0 ** (k - 1))


def test_oracle_gradients_are_the_formulas_and_match_differences():
    """dx = dy W and dW = dy^T x are the derivatives of <dy, x W^T>; quantisation is passed straight through."""
    rng = np.random.default_rng(5)
    x, w, dy = rng.standard_normal((6, 40)), rng.standard_normal((9, 40)), rng.standard_normal((6, 9))
    f = lambda a, b: (dy * (a @ b.T)).sum()   # noqa: E731
    vx, vw, s = rng.standard_normal(x.shape), rng.standard_normal(w.shape), 1e-5
    np.testing.assert_allclose(((dy @ w) * vx).sum(), (f(x + s * vx, w) - f(x - s * vx, w)) / (2 * s), rtol=1e-8)
    np.testing.assert_allclose(((dy.T @ x) * vw).sum(), (f(x, w + s * vw) - f(x, w - s * vw)) / (2 * s), rtol=1e-8)


def _cpu_weight(n, k):
    kp = (k + 127) // 128 * 128
    return (torch.zeros(n, kp, dtype=torch.uint8).view(torch.float8_e4m3fn),
            torch.full(((n + 127) // 128, kp // 128), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu))


def test_refusals():
    import yolo_from_scratch_amd as y
    d, s = _cpu_weight(40, 200)
    w = y.Fp8Tensor(d, s, 200)
    assert w.shape == (40, 200) and w.dequantize().shape == (40, 200)
    x, m = torch.zeros(3, 200), torch.zeros(40, 200)
    for call in (lambda: y.Fp8Tensor(d, s, 300), lambda: y.Fp8Tensor(d, s, 100), lambda: y.Fp8Tensor(d, s, 0),
                 lambda: y.Fp8Tensor(d, s, 200, (1, 128)), lambda: y.Fp8Tensor(d.float(), s, 200),
                 lambda: y.Fp8Tensor(d, s.view(torch.uint8), 200), lambda: y.Fp8Tensor(d, s[:, :1], 200),
                 lambda: y.Fp8Tensor(d[:, :128], s, 128), lambda: y.Fp8Tensor(d.view(-1), s, 200),
                 lambda: y.quantize_fp8(m), lambda: y.quantize_fp8(m[0]), lambda: y.quantize_fp8(m.double()),
                 lambda: y.quantize_fp8(torch.zeros(0, 8)), lambda: y.fp8_matmul(x, w), lambda: y.fp8_matmul(x, m),
                 lambda: y.fp8_matmul(x[:, :100], w), lambda: y.fp8_matmul(x.int(), w), lambda: y.fp8_matmul(torch.zeros(()), w),
                 lambda: y.fp8_matmul(x, w, torch.zeros(39)), lambda: y.fp8_matmul(x, w, torch.zeros(40).int()),
                 lambda: y.fp8_matmul(x, w, slope=-0.1), lambda: y.fp8_matmul(x, w, slope=2.0),
                 lambda: y.fp8_matmul(x, w, out_dtype=torch.float64), lambda: y.fp8_linear(x, m),
                 lambda: y.fp8_linear(x[:, :10], m), lambda: y.fp8_linear(x.long(), m), lambda: y.fp8_linear(x, m.double()),
                 lambda: y.fp8_linear(x, m, torch.zeros(41))):
        with pytest.raises(y.YfsError):
            call()


def test_refusals_of_the_library():
    import yolo_from_scratch_amd as y
    lib, p = y.lib(), 4096
    big = 1 << 23
    assert lib.yfs_fp8_gemm(p, p, p, p, 1, None, p, 1, 8, 8, 8, 1.0, 0, None, 0, None) == -2      # row scales on both sides: fp32 only
    assert lib.yfs_fp8_quantize_weight(None, 0, 8, 8, 8, p, p, None, None, None) == -1
    assert lib.yfs_fp8_quantize_weight(p, 0, 8, 8, 8, p, p, p, None, None) == -1
    assert lib.yfs_fp8_quantize_weight(p, 0, 8, big, 8, p, p, None, None, None) == -1
    assert lib.yfs_fp8_quantize_weight(p, 9, 8, 8, 8, p, p, None, None, None) == -2
    assert lib.yfs_fp8_quantize_weight(p, 0, 8, 8, 8, p + 8, p, None, None, None) == -1
    assert lib.yfs_fp8_quantize_rows(p, 0, 8, 8, 8, None, None, None, None, None, None) == -1
    assert lib.yfs_fp8_quantize_rows(p, 0, 8, 0, 8, p, p, None, None, None, None) == -1
    assert lib.yfs_fp8_gemm(p, p, p, p, 0, None, None, 1, 8, 8, 8, 1.0, 0, None, 0, None) == -1
    assert lib.yfs_fp8_gemm(p, p, p, p, 0, None, p, 1, 8, 8, 8, 1.0, 1, None, 0, None) == -2      # bf16 does not accumulate
    assert lib.yfs_fp8_gemm(p, p, p, p, 0, None, p, 1, 8, 8, 8, 3.0, 0, None, 0, None) == -1
    need = lib.yfs_fp8_gemm_workspace_bytes(64, 4096, 50176)
    assert need > 0 and lib.yfs_fp8_gemm(p, p, p, p, 0, None, p, 1, 64, 4096, 50176, 1.0, 0, p, need - 1, None) == -3
    need = lib.yfs_fp8_matmul_workspace_bytes(30, 40, 200)
    assert need > 0 and lib.yfs_fp8_matmul(p, 1, 200, p, p, None, p, 1, 30, 40, 200, 1.0, p, need - 1, None) == -3
    assert lib.yfs_fp8_matmul(p, 1, 200, p, p, None, p, 1, 30, 40, 200, 1.0, p + 16, need, None) == -3
    assert lib.yfs_fp8_matmul_workspace_bytes(0, 1, 1) == 0 and lib.yfs_fp8_gemm_workspace_bytes(1, big, 1) == 0
    assert lib.yfs_fp8_colsum(p, 0, 8, p, 0, None) == -1
    fwd, saved = lib.yfs_fp8_linear_fwd_workspace_bytes(5, 6, 7), lib.yfs_fp8_linear_saved_bytes(5, 6, 7, 3)
    bwd = lib.yfs_fp8_linear_bwd_workspace_bytes(5, 6, 7, 7)
    assert fwd and saved and bwd and lib.yfs_fp8_linear_saved_bytes(5, 6, 7, 0) == 0 and lib.yfs_fp8_linear_saved_bytes(0, 6, 7, 3) == 0
    call = lambda y, needs, sb, wb: lib.yfs_fp8_linear_fwd(p, 1, 7, p, 0, 7, None, y, 1, 5, 6, 7, needs, p, sb, p, wb, None)   # noqa: E731
    assert call(None, 3, saved, fwd) == -1 and call(p, 3, saved - 1, fwd) == -3 and call(p, 3, saved, fwd - 1) == -3
    back = lambda dx, dw, db, needs, wb: lib.yfs_fp8_linear_bwd(p, 1, 6, dx, 1, dw, 0, db, 0, 5, 6, 7, needs, p, 1 << 20, p, wb, None)   # noqa: E731
    assert back(p, p, None, 7, bwd) == -1 and back(None, p, p, 7, bwd) == -1 and back(None, None, p, 4, bwd) == -1
    assert back(p, p, p, 7, bwd - 1) == -3


def _quantize_rows(x, rows, cols, colsum=False):
    """yfs_fp8_quantize_rows: x by rows and / or its transpose by rows, with packed scales, and the tile column sums."""
    from yolo_from_scratch_amd import _lib as L
    (m, k), dev, lib = x.shape, x.device, L.lib()
    pad = lambda n: (n + 127) // 128 * 128   # noqa: E731
    e4, u8 = torch.float8_e4m3fn, torch.uint8
    q = torch.empty(m, pad(k), device=dev, dtype=e4) if rows else None
    s = torch.empty(lib.yfs_fp8_packed_scale_bytes(m, k), device=dev, dtype=u8) if rows else None
    qt = torch.empty(k, pad(m), device=dev, dtype=e4) if cols else None
    st = torch.empty(lib.yfs_fp8_packed_scale_bytes(k, m), device=dev, dtype=u8) if cols else None
    cs = torch.empty(pad(m) // 128, k, device=dev, dtype=torch.float32) if colsum else None
    p = lambda t: t.data_ptr() if t is not None else None   # noqa: E731
    L.check(lib.yfs_fp8_quantize_rows(x.data_ptr(), L.DTYPES[x.dtype], x.stride(0), m, k, p(q), p(s), p(qt), p(st), p(cs),
                                      torch.cuda.current_stream().cuda_stream), "yfs_fp8_quantize_rows")
    return q, s, qt, st, cs


# ---- GPU: quantisers -------------------------------------------------------------------------------------------------
def _unpack_scales(packed, rows, blocks):
    """Packed row scales -> exponents [rows, blocks]."""
    groups = (rows + 255) // 256 * 4
    t = packed.cpu().numpy().reshape(blocks, groups, 16, 4).transpose(0, 1, 3, 2).reshape(blocks, groups * 64)[:, :rows]
    return t.T.astype(np.int64) - 127


def _edge_values(rows, cols, dtype):
    """Blocks of zeros, of subnormals, at the upper end, on the border of a scale, with NaN and infinities."""
    t = _matrix(rows, cols, rows * 31 + cols, torch.float32, "cpu")
    flat = t.view(-1)
    flat[::7] = 448.0
    flat[1::11] = 0.0
    t[:, : min(3, cols)] *= 2.0 ** -20
    if rows > 4:
        t[1] = 0.0
        t[2] = t[2] * 2.0 ** -120 if dtype != torch.float16 else t[2] * 2.0 ** -14
        t[3] = t[3] * 2.0 ** 100 if dtype != torch.float16 else t[3]
        t[4, 0], t[4, -1] = float("nan"), float("inf")
    return t.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (5, 8), (16, 300), (127, 64), (128, 128), (129, 257), (300, 520)])
def test_quantisers(rows, cols, dtype):
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import fp8_ops as f8
    x = _edge_values(rows, cols, DTYPES[dtype])
    xn = x.double().numpy()
    xd = x.to(DEV)
    wide = torch.zeros(rows, cols + 9, dtype=x.dtype, device=DEV)
    wide[:, 5:5 + cols] = xd
    for src in (xd, wide[:, 5:5 + cols]):                    # dense, and rows at odd offsets with a stride of their own
        q, s, qt, st, cs = _quantize_rows(src, True, True, True)
        kb, mb = (cols + 127) // 128, (rows + 127) // 128
        for got, packed, arr, n, blocks in ((q, s, xn, rows, kb), (qt, st, xn.T, cols, mb)):
            ref, e = hr.quantize(arr, 1, 128)
            assert np.array_equal(_unpack_scales(packed, n, blocks), e)
            vals = _np(got.float())
            assert np.array_equal(vals[:, : arr.shape[1]], ref, equal_nan=True) and (vals[:, arr.shape[1]:] == 0).all()
        alone = _quantize_rows(src, True, False)[0], _quantize_rows(src, False, True)[2]
        assert torch.equal(alone[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(alone[1].view(torch.uint8), qt.view(torch.uint8))
        finite = np.isfinite(xn).all(0)
        _close(_np(cs.double().sum(0))[finite], xn.sum(0)[finite], (128 * 2.0 ** -24 * np.abs(xn).sum(0) + 1e-40)[finite], "column sums")
        wq, ws, wqt, wst = f8._quantize_weight(src, True)
        ref, e = hr.quantize(xn, 128, 128)
        assert np.array_equal(ws.view(torch.uint8).cpu().numpy().astype(np.int64) - 127, e)
        assert np.array_equal(_np(wq.float())[:, :cols], ref, equal_nan=True)
        assert np.array_equal(_np(wqt.float())[:, :rows], ref.T, equal_nan=True) and torch.equal(wst.view(torch.uint8), ws.view(torch.uint8).t())
        t = yfs.quantize_fp8(src)
        assert torch.equal(t.data.view(torch.uint8), wq.view(torch.uint8))
        assert np.array_equal(_np(t.dequantize()), hr.rounded(xn, 128, 128).astype(np.float32).astype(np.float64), equal_nan=True)


# ---- GPU: products ---------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 3, 5), (1, 1470, 4096), (2, 16, 128), (3, 100, 129), (7, 257, 1000), (15, 64, 64), (16, 128, 256),
          (17, 129, 127), (31, 40, 3000), (33, 300, 384), (63, 65, 640), (64, 256, 1024), (65, 17, 130), (127, 130, 260),
          (128, 128, 128), (129, 255, 385), (200, 384, 512), (257, 513, 700), (300, 20, 2048), (20, 1000, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(m, n, k):
    import yolo_from_scratch_amd as yfs
    w = _matrix(n, k, n + k)
    wq = yfs.quantize_fp8(w)
    bias = torch.randn(n, device=DEV)
    wn, bn = hr.rounded(_np(w), 128, 128), _np(bias)
    for name, t in DTYPES.items():
        x = _matrix(m, k, 3 * m + k, t)
        if t == torch.float16:
            x = x.clamp(-1000, 1000)
        xn = hr.rounded(_np(x), 1, 128)
        plain = xn @ wn.T
        for out in DTYPES.values():
            if out == torch.float16 and np.abs(plain).max() > 60000:
                continue
            got = yfs.fp8_matmul(x, wq, out_dtype=out)
            assert got.dtype == out and got.shape == (m, n)
            _close(_np(got), plain, _tolerance(xn, wn, plain, out), f"{name} -> {out}")
        ref = plain + bn
        got = yfs.fp8_matmul(x, wq, bias, 0.1, torch.bfloat16)
        tol = _tolerance(xn, wn, ref, torch.bfloat16, bn)
        _close(_np(got), np.where(ref > 0, ref, 0.1 * ref), tol * np.where(np.abs(ref) <= tol, 2.0, 1.01), "bias and slope")
        assert torch.equal(got, yfs.fp8_matmul(x, wq, bias, 0.1, torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,kernel", [(1, 4096, 50176, "fp8_rows_kernel"), (3, 40, 50176, "fp8_rows_kernel"),
                                          (16, 1470, 4096, "fp8_rows_kernel"), (16, 512, 50176, "fp8_gemm_kernel<64,128,splits"),
                                          (64, 512, 50176, "fp8_gemm_kernel<64,128,splits"), (3, 70000, 300, "fp8_rows_kernel"),
                                          (20, 40000, 300, "fp8_gemm_kernel<64,128,splits1>"),
                                          (300, 2600, 1111, "fp8_gemm_kernel<64,64,splits1>"),
                                          (1500, 1300, 1111, "fp8_gemm_kernel<64,128,splits1>"),
                                          (2600, 2900, 500, "fp8_gemm_kernel<128,128,splits1>"),
                                          (3000, 4096, 515, "fp8_gemm8_kernel<rest0>"), (4099, 4101, 640, "fp8_gemm8_kernel<rest259>"),
                                          (4352, 4096, 768, "fp8_gemm8_kernel<rest256>"), (2100, 8300, 515, "fp8_gemm8_kernel<rest308>"),
                                          (16300, 1100, 257, "fp8_gemm8_kernel<rest"), (8192, 2304, 2048, "fp8_gemm8_kernel")])
def test_matmul_large_against_fp64_on_the_gpu(m, n, k, kernel):
    """Every kernel the size rule chooses, at ragged sizes and odd counts of blocks."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import _lib as L
    g = torch.Generator(DEV).manual_seed(m + n)
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    w = torch.randn(n, k, device=DEV, generator=g) / k ** 0.5
    wq = yfs.quantize_fp8(w)
    xn = torch.from_numpy(hr.rounded(_np(x), 1, 128)).to(DEV)
    wd = wq.dequantize().double()
    ref = xn @ wd.t()
    mag = xn.abs() @ wd.abs().t()
    f32 = yfs.fp8_matmul(x, wq, out_dtype=torch.float32).double()
    assert ((f32 - ref).abs() <= (96 + k / 32) * 2.0 ** -24 * mag).all()
    assert float((f32 - ref).norm() / ref.norm()) < 2e-6
    b16 = yfs.fp8_matmul(x, wq).double()
    assert L.last_kernel().startswith(kernel)
    assert float((b16 - ref).norm() / ref.norm()) < 2.0 ** -8      # every value within half a step, 2^-8 of it at most
    assert float((b16 - f32.bfloat16().double()).norm() / ref.norm()) < 2.0 ** -9


@pytest.mark.gpu
def test_shapes_strides_and_special_values():
    import yolo_from_scratch_amd as yfs
    w = _matrix(70, 200, 9)
    wq = yfs.quantize_fp8(w)
    wide = _matrix(48, 420, 10, torch.bfloat16)
    for x in (wide[:, 3:203], wide[::2, 100:300], wide[:4, :200].view(2, 2, 200), wide[7, 1:201], wide[:1, :200].expand(5, 200),
              _matrix(200, 33, 11, torch.bfloat16).t()):
        got = yfs.fp8_matmul(x, wq)
        assert got.shape == x.shape[:-1] + (70,)
        assert torch.equal(got.reshape(-1, 70), yfs.fp8_matmul(x.reshape(-1, 200).contiguous(), wq))
    assert yfs.fp8_matmul(wide[:0, :200], wq).shape == (0, 70)
    clean = _matrix(20, 200, 12, torch.bfloat16)
    y0 = yfs.fp8_matmul(clean, wq)
    x = clean.clone()
    x[3, 5], x[9, 199], x[19, 130] = float("nan"), float("inf"), -float("inf")
    y = yfs.fp8_matmul(x, wq)
    bad = torch.zeros(20, dtype=torch.bool, device=DEV)
    bad[[3, 9, 19]] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], y0[~bad])
    wn = w.clone()
    wn[11, 150] = float("nan")
    y = yfs.fp8_matmul(clean, yfs.quantize_fp8(wn))
    assert y[:, 11].isnan().all() and torch.equal(y[:, torch.arange(70, device=DEV) != 11], y0[:, torch.arange(70, device=DEV) != 11])
    assert (yfs.fp8_matmul(torch.zeros_like(clean), wq) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 40, 200), (5, 129, 64), (64, 100, 300), (128, 128, 128), (130, 257, 131), (300, 64, 513),
                                   (40, 1300, 1500), (600, 1500, 1400)])
def test_linear_forward_and_gradients(m, n, k, dtype):
    import yolo_from_scratch_amd as yfs
    t = DTYPES[dtype]
    x = _matrix(m, k, m + k, t).clamp(-100, 100)
    w = _matrix(n, k, n + 2 * k) / 64
    b = torch.randn(n, device=DEV)
    dy = (_matrix(m, n, 5 * m + n) / 64).to(t).clamp(-100, 100)
    for v in (x, w, b):
        v.requires_grad_()
    y = yfs.fp8_linear(x, w, b)
    assert y.dtype == t
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dx.dtype == t and dw.dtype == torch.float32 and db.dtype == torch.float32
    xn, wn, dyn, bn = _np(x), _np(w), _np(dy), _np(b)
    xq, wq, dq = hr.rounded(xn, 1, 128), hr.rounded(wn, 128, 128), hr.rounded(dyn, 1, 128)
    ref = xq @ wq.T + bn
    _close(_np(y), ref, _tolerance(xq, wq, ref, t, bn), "y")
    ref = dq @ wq
    _close(_np(dx), ref, _tolerance(dq, wq.T, ref, t), "dx")
    xt, dt = hr.rounded(xn.T, 1, 128), hr.rounded(dyn.T, 1, 128)
    ref = dt @ xt.T
    _close(_np(dw), ref, _tolerance(dt, xt, ref, torch.float32), "dw")
    _close(_np(db), dyn.sum(0), (128 + m) * 2.0 ** -24 * np.abs(dyn).sum(0) + 1e-37, "db")
    # some of the gradients alone are the same numbers
    only_w, = torch.autograd.grad(yfs.fp8_linear(x.detach(), w), w, dy)
    assert torch.equal(only_w, dw)
    only_x, = torch.autograd.grad(yfs.fp8_linear(x, w.detach()), x, dy)
    assert torch.equal(only_x, dx)
    only_b, = torch.autograd.grad(yfs.fp8_linear(x.detach(), w.detach(), b), b, dy)
    _close(_np(only_b), dyn.sum(0), (128 + m) * 2.0 ** -24 * np.abs(dyn).sum(0) + 1e-37, "db alone")


@pytest.mark.gpu
def test_linear_other_shapes():
    import yolo_from_scratch_amd as yfs
    w = (_matrix(40, 96, 1) / 16).requires_grad_()
    x = _matrix(60, 96, 2, torch.bfloat16).view(3, 4, 5, 96).requires_grad_()
    y = yfs.fp8_linear(x, w)
    assert y.shape == (3, 4, 5, 40)
    gx, gw = torch.autograd.grad(y.float().sum(), (x, w))            # an expanded gradient
    flat = x.detach().view(60, 96).requires_grad_()
    fx, fw = torch.autograd.grad(yfs.fp8_linear(flat, w), (flat, w), torch.ones(60, 40, device=DEV, dtype=torch.bfloat16))
    assert torch.equal(gx.view(60, 96), fx) and torch.equal(gw, fw)
    e = torch.empty(0, 96, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    ge, gw = torch.autograd.grad(yfs.fp8_linear(e, w).sum(), (e, w))
    assert ge.shape == (0, 96) and (gw == 0).all() and gw.shape == w.shape
    wh = w.detach().bfloat16().requires_grad_()
    gw, = torch.autograd.grad(yfs.fp8_linear(flat.detach(), wh), wh, torch.ones(60, 40, device=DEV, dtype=torch.bfloat16))
    assert gw.dtype == torch.bfloat16


@pytest.mark.gpu
def test_gradients_against_differences():
    """Straight through the quantisers: with operands that 8 bits hold exactly (whole numbers to 8), f is bilinear, and the
    central difference along a direction of such numbers is exact up to fp32 sums."""
    import yolo_from_scratch_amd as yfs
    g = torch.Generator().manual_seed(4)
    ints = lambda *s: torch.randint(-4, 5, s, generator=g).float().to(DEV)   # noqa: E731
    x, w, vx, vw, dy = ints(40, 200), ints(70, 200), ints(40, 200), ints(70, 200), ints(40, 70)
    x[:, ::128], w[::128, ::128], dy[:, 0] = 4.0, 4.0, 4.0
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(yfs.fp8_linear(x, w), (x, w), dy)
    f = lambda a, b: float((yfs.fp8_linear(a, b).double() * dy.double()).sum())   # noqa: E731
    with torch.no_grad():
        assert float((dx.double() * vx.double()).sum()) == (f(x + vx, w) - f(x - vx, w)) / 2
        assert float((dw.double() * vw.double()).sum()) == (f(x, w + vw) - f(x, w - vw)) / 2


@pytest.mark.gpu
def test_nothing_is_written_outside():
    from yolo_from_scratch_amd import _lib as L
    from yolo_from_scratch_amd import fp8_ops as f8
    lib, s = L.lib(), torch.cuda.current_stream().cuda_stream
    for m, n, k, out in ((5, 130, 300, torch.bfloat16), (70, 33, 2048, torch.float32), (130, 131, 129, torch.float16)):
        x, w = _matrix(m, k, 1, torch.bfloat16).clamp(-8, 8), _matrix(n, k, 2) / 1000
        wq, ws, _, _ = f8._quantize_weight(w, False)
        need = lib.yfs_fp8_matmul_workspace_bytes(m, n, k)
        space = torch.full((need + 512,), 77, device=DEV, dtype=torch.uint8)
        space = space[(-space.data_ptr()) % 256:]
        y = torch.full((m * n + 64,), 3.0, device=DEV, dtype=out)
        L.check(lib.yfs_fp8_matmul(x.data_ptr(), 1, k, wq.data_ptr(), ws.data_ptr(), None, y.data_ptr(), L.DTYPES[out], m, n, k, 1.0,
                                   space.data_ptr(), need, s), "matmul")
        assert (y[m * n:] == 3).all() and (space[need:] == 77).all()
        ref = hr.rounded(_np(x), 1, 128) @ hr.rounded(_np(w), 128, 128).T
        _close(_np(y[: m * n]).reshape(m, n), ref, _tolerance(hr.rounded(_np(x), 1, 128), hr.rounded(_np(w), 128, 128), ref, out), "y")
        kp, mp = (k + 127) // 128 * 128, (m + 127) // 128 * 128
        sizes = (m * kp, lib.yfs_fp8_packed_scale_bytes(m, k), k * mp, lib.yfs_fp8_packed_scale_bytes(k, m))
        bufs = [torch.full((v + 256,), 77, device=DEV, dtype=torch.uint8) for v in sizes]
        L.check(lib.yfs_fp8_quantize_rows(x.data_ptr(), 1, k, m, k, *[v.data_ptr() for v in bufs], None, s), "quantize")
        for v, size in zip(bufs, sizes):
            assert (v[size:] == 77).all()


@pytest.mark.gpu
def test_other_stream_and_captured_graphs():
    """Forward and backward on another stream, and two captured graphs replayed in turn between eager work."""
    import yolo_from_scratch_amd as yfs
    x = _matrix(70, 1000, 1, torch.bfloat16).requires_grad_()
    w = (_matrix(300, 1000, 2) / 32).requires_grad_()
    b = torch.randn(300, device=DEV).requires_grad_()
    dy = _matrix(70, 300, 3, torch.bfloat16)

    def step():
        y = yfs.fp8_linear(x, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    frozen = yfs.quantize_fp8(w)

    def serve():
        return (yfs.fp8_matmul(x, frozen, b, 0.1), yfs.fp8_matmul(x[:1], frozen))
    want, want2 = step(), serve()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        serve()
        ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(ga, stream=side):
            out = step()
        with torch.cuda.graph(gb, stream=side):
            out2 = serve()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.roll(x, 3, 0) * 0.5)
            w.mul_(1.5)
        want, want2 = step(), serve()
        for t in out + out2:
            t.fill_(9)
        ga.replay(), gb.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out + out2, want + want2)), k


@pytest.mark.gpu
def test_module_with_flat_sgd():
    """Fp8Linear's gradients reach FlatSGD's arena directly: the same numbers as without it, also over two backward passes."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd.train import FlatSGD
    torch.manual_seed(2)
    lin = yfs.Fp8Linear(300, 140).to(DEV)
    assert list(lin.state_dict()) == ["weight", "bias"]
    x = [torch.randn(90, 300, device=DEV) for _ in range(2)]
    want = []
    for v in x:
        want.append(torch.autograd.grad(lin(v).float().square().sum(), (lin.weight, lin.bias)))
    opt = FlatSGD(lin.parameters(), lr=0.01, momentum=0.9)
    before = lin.weight.detach().clone()
    opt.zero_grad()
    lin(x[0]).float().square().sum().backward()
    assert torch.equal(lin.weight.grad, want[0][0]) and torch.equal(lin.bias.grad, want[0][1])
    lin(x[1]).float().square().sum().backward()
    for p, q, r in zip((lin.weight.grad, lin.bias.grad), want[0], want[1]):
        assert float((p - (q + r)).abs().max()) <= 2.0 ** -22 * float((q.abs() + r.abs()).max())
    opt.step(max_norm=None)
    assert not torch.equal(lin.weight, before)
    opt.zero_grad()
    lin(x[1]).float().square().sum().backward()                     # fresh again: overwritten, with the moved weights
    assert torch.isfinite(lin.weight.grad).all()


@pytest.mark.gpu
def test_frozen_layers():
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import model as ym
    net = torch.nn.Sequential(ym.HipLinear(200, 96, fused_act=0.1), torch.nn.Identity(), torch.nn.Sequential(torch.nn.Linear(96, 10))).to(DEV)
    x = torch.randn(5, 200, device=DEV)
    want = torch.nn.functional.leaky_relu(yfs.fp8_matmul(x, yfs.quantize_fp8(net[0].weight), net[0].bias, out_dtype=torch.float32), 0.1).bfloat16()
    last = net[2][0]
    want = yfs.fp8_matmul(want, yfs.quantize_fp8(last.weight), last.bias, out_dtype=torch.float32)
    frozen = yfs.freeze_fp8(net)
    assert frozen is net and not list(net.parameters()) and not net.training
    got = net(x)
    assert got.dtype == torch.bfloat16
    # the hidden value is rounded from 8-bit-instruction sums here, from fp32 sums above: at most a step of bf16 apart, 2^-7,
    # so its 8-bit rounding differs by a step (2^-3) at most where it crosses a border
    assert float((got.float() - want).abs().max()) < 2.0 ** -3 * float(want.abs().max())
    state = {k: v.clone() for k, v in net.state_dict().items()}
    net.load_state_dict(state)
    assert torch.equal(net(x), got)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(5, 300), (20, 300), (300, 200)])
def test_smallest_scales(m, k):
    """Blocks around the smallest scale, 2^-127, and below it.  A widened operand is off by half the smallest bf16, 2^-134, at most."""
    import yolo_from_scratch_amd as yfs
    x = _matrix(m, k, 21, device="cpu")
    for i, e in enumerate((-118, -122, -126, -130, -136)):
        x[i::5] *= 2.0 ** e / x[i::5].abs().amax(1, keepdim=True)
    x[:, 128:] *= 2.0 ** -3
    x = x.to(DEV)
    w = _matrix(70, k, 22) * 2.0 ** 100
    wq = yfs.quantize_fp8(w)
    xn, wn = hr.rounded(_np(x), 1, 128), hr.rounded(_np(w), 128, 128)
    ref = xn @ wn.T
    for out in (torch.float32, torch.bfloat16):
        tol = _tolerance(xn, wn, ref, out)
        if out == torch.float32:
            tol = tol + 2.0 ** -134 * np.abs(wn).sum(1)
        _close(_np(yfs.fp8_matmul(x, wq, out_dtype=out)), ref, tol, str(out))


@pytest.mark.gpu
def test_serving_a_layer_that_trains_keeps_nothing():
    """A layer bound to an optimiser's arena, called without gradients, does what fp8_linear of plain tensors does."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd.train import FlatSGD
    lin = yfs.Fp8Linear(300, 70).to(DEV)
    x = _matrix(33, 300, 23, torch.bfloat16)
    FlatSGD(lin.parameters(), lr=0.1)
    with torch.no_grad():
        y = lin(x)
        assert y.grad_fn is None and torch.equal(y, yfs.fp8_linear(x, lin.weight.clone(), lin.bias.clone()))
    assert torch.equal(lin(x), y)


def test_freeze_refuses_a_layer_alone():
    import yolo_from_scratch_amd as yfs
    with pytest.raises(yfs.YfsError, match="FrozenFp8Linear"):
        yfs.freeze_fp8(torch.nn.Linear(4, 4))


@pytest.mark.gpu
def test_freeze_converts_a_shared_layer_once_and_all_or_none():
    import yolo_from_scratch_amd as yfs
    lin = torch.nn.Linear(64, 64).to(DEV)
    net = torch.nn.Sequential(lin, torch.nn.ReLU(), lin, torch.nn.Sequential(lin))
    yfs.freeze_fp8(net)
    assert isinstance(net[0], yfs.FrozenFp8Linear) and net[2] is net[0] and net[3][0] is net[0]
    net = torch.nn.Sequential(torch.nn.Linear(8, 8).to(DEV), torch.nn.Linear(8, 8).double().to(DEV))
    with pytest.raises(yfs.YfsError):
        yfs.freeze_fp8(net)
    assert isinstance(net[0], torch.nn.Linear) and net.training


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(64, 300, 1000), (65, 300, 1000), (1, 4096, 4096), (33, 1, 50176), (64, 40, 50176), (17, 1470, 130)])
def test_linear_around_the_rows_that_are_quantised_in_the_product(m, n, k):
    """Up to 64 rows the weights are quantised by the workgroups that multiply them: the forward pass is that of stored weights,
    to the rounding of the output, with and without gradients, and the transposed operands are those of the other form."""
    import yolo_from_scratch_amd as yfs
    x, w, b = _matrix(m, k, 31, torch.bfloat16), _matrix(n, k, 32), torch.randn(n, device=DEV)
    dy = _matrix(m, n, 33, torch.bfloat16)
    xn, wn, dn = hr.rounded(_np(x), 1, 128), hr.rounded(_np(w), 128, 128), hr.rounded(_np(dy), 1, 128)
    ref = xn @ wn.T + _np(b)
    for wt in (w, w.bfloat16(), w.half()):
        wr = wn if wt is w else hr.rounded(_np(wt), 128, 128)
        r = ref if wt is w else xn @ wr.T + _np(b)
        y = yfs.fp8_linear(x, wt, b)
        _close(_np(y), r, _tolerance(xn, wr, r, torch.bfloat16, _np(b)), f"y, {wt.dtype} weights")
    y32 = yfs.fp8_linear(x.float(), w, b)
    _close(_np(y32), ref, _tolerance(xn, wn, ref, torch.float32, _np(b)), "fp32 y")
    x, w = x.requires_grad_(), w.requires_grad_()
    y = yfs.fp8_linear(x, w, b)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    _close(_np(y), ref, _tolerance(xn, wn, ref, torch.bfloat16, _np(b)), "y")
    plain = dn @ wn
    _close(_np(dx), plain, _tolerance(dn, wn.T, plain, torch.bfloat16), "dx")
    dt, xt = hr.rounded(_np(dy).T, 1, 128), hr.rounded(_np(x).T, 1, 128)
    plain = dt @ xt.T
    _close(_np(dw), plain, _tolerance(dt, xt, plain, torch.float32), "dw")
    only = torch.autograd.grad(yfs.fp8_linear(x, w.detach(), b), x, dy)[0]
    assert torch.equal(only, dx)
    only = torch.autograd.grad(yfs.fp8_linear(x.detach(), w, b), w, dy)[0]
    assert torch.equal(only, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [30011, 30016])
def test_large_weights_that_pass_the_caches_by(k):
    """From 128 MiB on weights are read and their gradients written past the caches where rows begin on a line of 128 bytes: the
    same values as in parts below that size."""
    import yolo_from_scratch_amd as yfs
    n = 1160                              # 139 MB
    w = _matrix(n, k, 41).requires_grad_()
    for m in (40, 200):
        x, dy = _matrix(m, k, 42, torch.bfloat16), _matrix(m, n, 43, torch.bfloat16)
        y = yfs.fp8_linear(x, w)
        dw, = torch.autograd.grad(y, w, dy)
        for lo, hi in ((0, 640), (640, 1160)):
            part = w.detach()[lo:hi].contiguous().requires_grad_()
            yp = yfs.fp8_linear(x, part)
            dp, = torch.autograd.grad(yp, part, dy[:, lo:hi].contiguous())
            # the reduction is split by the count of columns, so y may be rounded the other way
            assert torch.equal(dp, dw[lo:hi]) and float((yp.float() - y[:, lo:hi].float()).detach().abs().max()) <= 2.0 ** -7 * float(y.detach().abs().max())
    from yolo_from_scratch_amd.train import FlatSGD
    lin = yfs.Fp8Linear(k, n, bias=False).to(DEV)
    with torch.no_grad():
        lin.weight.copy_(w)
    FlatSGD(lin.parameters(), lr=0.1)
    lin(x).backward(dy)
    assert torch.equal(lin.weight.grad, dw)
    lin(x).backward(dy)
    assert torch.equal(lin.weight.grad, dw + dw)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(300, 1400, 16500), (129, 3970, 16400), (260, 4000, 8200), (200, 28000, 300), (140, 34000, 200), (130, 26000, 260)])
def test_each_split_and_tile_of_mid_sized_products(m, n, k):
    """Split 128 x 128 and 64 x 128 tiles, one round of 256 x 256 tiles that are not full: 16-bit and 32-bit outputs."""
    import yolo_from_scratch_amd as yfs
    x, w = _matrix(m, k, 51, torch.bfloat16), _matrix(n, k, 52)
    wq = yfs.quantize_fp8(w)
    xn, wn = hr.rounded(_np(x), 1, 128), wq.dequantize().double()
    xg = torch.from_numpy(xn).to(DEV)
    ref, mag = xg @ wn.t(), xg.abs() @ wn.abs().t()
    inner = (96 + k / 32) * 2.0 ** -24 * mag
    got = yfs.fp8_matmul(x, wq, out_dtype=torch.float32).double()
    assert bool(((got - ref).abs() <= 2.0 ** -24 * (ref.abs() + inner) + inner).all())
    # the 8-bit instruction: 2^-9 of the largest product of each block of 128
    for k0 in range(0, k, 128):
        inner = inner + 2.0 ** -9 * xg[:, k0:k0 + 128].abs().amax(1, keepdim=True) * wn[:, k0:k0 + 128].abs().amax(1)
    got = yfs.fp8_matmul(x, wq).double()
    assert bool(((got - ref).abs() <= 2.0 ** -8 * (ref.abs() + inner) + inner).all())
    assert torch.equal(yfs.fp8_matmul(x, wq).double(), got)


def _plan(m, n, k, dtype):
    import ctypes
    import yolo_from_scratch_amd as y
    from yolo_from_scratch_amd import _lib as L
    plan = (ctypes.c_int64 * 5)()
    assert y.lib().yfs_fp8_gemm_plan(m, n, k, L.DTYPES[dtype], ctypes.addressof(plan)) == 0
    return tuple(plan)


def test_plan_covers_every_product():
    """Every launch that a plan stands for has workgroups: 256 x 256 tiles have rows to take wherever they are chosen, in whole
    tiles or to the end, and every part of a split reduction has blocks."""
    import random
    rng = random.Random(7)
    size = lambda top: max(1, min(top, int(2 ** rng.uniform(0, np.log2(top + 1)))))   # noqa: E731
    cases = [(size(1 << 15), size(1 << 18), size(1 << 17)) for _ in range(20000)]
    # one row of 256-wide tiles in one round and a bit more
    cases += [(m, n, k) for m in (192, 193, 200, 255, 256, 257) for n in (65536, 65537, 66000, 76800, 82944, 98304, 98305, 131072, 131073, 152064, 163840)
              for k in (64, 4096)]
    for m, n, k in cases:
        for t in (torch.bfloat16, torch.float32):
            bm, bn, parts, per, body = _plan(m, n, k, t)
            blocks = -(-k // 128)
            assert (bm, bn) in ((256, 256), (128, 128), (64, 128), (64, 64)), (m, n, k)
            assert parts >= 1 and (parts - 1) * per < blocks <= parts * per, (m, n, k)
            if bm == 256:
                assert t != torch.float32 and parts == 1 and (0 < body < m and body % 256 == 0 or body == m), (m, n, k, body)
            else:
                assert body == 0


def test_plan_refusals():
    import yolo_from_scratch_amd as y
    lib, p = y.lib(), 4096
    assert lib.yfs_fp8_gemm_plan(8, 8, 8, 1, None) == -1 and lib.yfs_fp8_gemm_plan(0, 8, 8, 1, p) == -1
    assert lib.yfs_fp8_gemm_plan(8, 8, 8, 7, p) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(256, 66000, 300), (200, 82944, 130), (193, 65537, 64), (256, 131073, 140)])
def test_one_row_of_tiles_wider_than_the_whole_rounds(m, n, k):
    import yolo_from_scratch_amd as yfs
    x, w = _matrix(m, k, 61, torch.bfloat16), _matrix(n, k, 62)
    wq = yfs.quantize_fp8(w)
    xg, wn = torch.from_numpy(hr.rounded(_np(x), 1, 128)).to(DEV), wq.dequantize().double()
    ref = xg @ wn.t()
    inner = (96 + k / 32) * 2.0 ** -24 * (xg.abs() @ wn.abs().t())
    for k0 in range(0, k, 128):       # the 8-bit instruction: 2^-9 of the largest product of each block of 128
        inner = inner + 2.0 ** -9 * xg[:, k0:k0 + 128].abs().amax(1, keepdim=True) * wn[:, k0:k0 + 128].abs().amax(1)
    got = yfs.fp8_matmul(x, wq).double()
    assert bool(((got - ref).abs() <= 2.0 ** -8 * (ref.abs() + inner) + inner).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [193, 200, 256])
def test_gradients_of_a_layer_with_more_than_65536_inputs(m):
    """dx of the head's first layer at 576 x 576 images: 82944 inputs."""
    import yolo_from_scratch_amd as yfs
    n, k = 130, 82944
    x = _matrix(m, k, 63, torch.bfloat16).requires_grad_()
    w = _matrix(n, k, 64).requires_grad_()
    dy = _matrix(m, n, 65, torch.bfloat16)
    dx, dw = torch.autograd.grad(yfs.fp8_linear(x, w), (x, w), dy)
    assert torch.isfinite(dw).all()
    dq, wq = torch.from_numpy(hr.rounded(_np(dy), 1, 128)).to(DEV), yfs.quantize_fp8(w).dequantize().double()
    ref = dq @ wq
    inner = (96 + n / 32) * 2.0 ** -24 * (dq.abs() @ wq.abs())
    for n0 in range(0, n, 128):
        inner = inner + 2.0 ** -9 * dq[:, n0:n0 + 128].abs().amax(1, keepdim=True) * wq[n0:n0 + 128].abs().amax(0)
    assert bool(((dx.double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + inner) + inner).all())


def test_a_step_that_is_still_running_is_waited_for(monkeypatch):
    """A weight whose overlapped optimiser step (FlatSGD.overlap_tail) may still be running is waited for before it is read:
    by the quantiser, a frozen layer and the product, in that order."""
    from yolo_from_scratch_amd import _lib as L
    from yolo_from_scratch_amd import fp8_ops as f8
    seen = []

    class Owner:
        def join(self):
            seen.append("join")

    class Ext:
        def fp8_linear(self, *a):
            seen.append("read")

        fp8_linear_check = fp8_linear

    def quantize(w, transposed):
        seen.append("read")
        return _cpu_weight(*w.shape) + (None, None)
    lin = torch.nn.Linear(200, 40)
    lin.weight._yfs_tail_owner, lin.weight._yfs_grad_sink = Owner(), torch.zeros(40, 200)
    monkeypatch.setattr(f8, "_quantize_weight", quantize)
    monkeypatch.setattr(L, "require_cuda", lambda *t: None)
    monkeypatch.setattr(L, "_binding", Ext())
    monkeypatch.setattr(f8._SinkLinearFn, "apply", lambda *a: seen.append("read"))
    f8.quantize_fp8(lin.weight)
    assert seen == ["join", "read"]
    f8.FrozenFp8Linear(lin)
    assert seen == ["join", "read"] * 2
    with torch.no_grad():
        f8.fp8_linear(torch.zeros(3, 200), lin.weight)
    assert seen == ["join", "read"] * 3
    f8.fp8_linear(torch.zeros(3, 200), lin.weight)
    assert seen == ["join", "read"] * 4 or seen == ["join", "read"] * 3 + ["join", "read", "read"]


@pytest.mark.gpu
def test_quantising_behind_an_overlapped_step():
    """The step of a large layer runs on a side stream; what is quantised right behind it is the weight after the step."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import model as ym
    from yolo_from_scratch_amd.train import FlatSGD
    torch.manual_seed(6)
    lin = ym.HipLinear(8192, 4096).to(DEV)
    opt = FlatSGD(lin.parameters(), lr=0.5, momentum=0.9, overlap_tail=True)
    x = torch.randn(64, 8192, device=DEV)
    for _ in range(3):
        opt.zero_grad()
        lin(x).float().square().mean().backward()
        opt.step(max_norm=None)
        assert opt._tail is not None
        q, frozen = yfs.quantize_fp8(lin.weight), yfs.FrozenFp8Linear(lin)
        torch.cuda.synchronize()
        want = yfs.quantize_fp8(lin.weight)
        for got in (q.data, frozen.weight_data):
            assert torch.equal(got.view(torch.uint8), want.data.view(torch.uint8))


def test_packed_scales_must_be_aligned():
    """The packed scales are fetched in dwords straight into LDS: q arrays and packed scales are 16-byte aligned, on both sides of
    a product and in the quantiser."""
    import yolo_from_scratch_amd as y
    lib, p = y.lib(), 4096
    gemm = lambda a, sa, b, sb, rows: lib.yfs_fp8_gemm(a, sa, b, sb, rows, None, p, 0, 8, 8, 8, 1.0, 1, None, 0, None)   # noqa: E731
    for bad in range(4):
        args = [p + 2 if i == bad else p for i in range(4)]
        assert gemm(*args, 1) == -1
    for off in (1, 8):
        assert lib.yfs_fp8_quantize_rows(p, 0, 8, 8, 8, p, p + off, None, None, None, None) == -1
        assert lib.yfs_fp8_quantize_rows(p, 0, 8, 8, 8, None, None, p, p + off, None, None) == -1


@pytest.mark.gpu
def test_backward_through_a_stored_weight_is_refused():
    """fp8_matmul has no gradient: a backward pass that reaches it says so, instead of leaving out what lies in front of it."""
    import yolo_from_scratch_amd as yfs
    wq = yfs.quantize_fp8(_matrix(40, 200, 71))
    frozen = yfs.FrozenFp8Linear(torch.nn.Linear(200, 40).to(DEV))
    front = _matrix(20, 200, 72).requires_grad_()
    bias = torch.randn(40, device=DEV, requires_grad=True)
    h = (2 * front).bfloat16()
    for y in (yfs.fp8_matmul(h, wq), frozen(h), yfs.fp8_matmul(h.detach(), wq, bias), yfs.fp8_matmul(front, wq), yfs.fp8_matmul(h[:0], wq)):
        loss = y.float().sum() + front.sum() + bias.sum()
        with pytest.raises(RuntimeError, match="fp8_matmul.*not differentiable"):
            loss.backward()
    with torch.no_grad():
        assert yfs.fp8_matmul(h, wq).grad_fn is None
    assert yfs.fp8_matmul(h.detach(), wq, bias.detach()).grad_fn is None and not frozen(h.detach()).requires_grad
    assert torch.equal(yfs.fp8_matmul(h, wq), yfs.fp8_matmul(h.detach(), wq))


@pytest.mark.gpu
def test_two_backward_passes_over_a_retained_graph():
    """A layer bound to an optimiser's arena takes several backward passes over one graph, as any other does: twice the gradient,
    which is exact, and the same dx."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd.train import FlatSGD
    torch.manual_seed(11)
    for bias in (True, False):
        lin = yfs.Fp8Linear(300, 140, bias=bias).to(DEV)
        opt = FlatSGD(lin.parameters(), lr=0.01, momentum=0.9)
        x = torch.randn(90, 300, device=DEV, requires_grad=True)
        opt.zero_grad()
        loss = lin(x).float().square().sum()
        loss.backward(retain_graph=True)
        once = [p.grad.clone() for p in (x, *lin.parameters())]
        loss.backward()
        for p, g in zip((x, *lin.parameters()), once):
            assert torch.equal(p.grad, g + g)


@pytest.mark.gpu
@pytest.mark.parametrize("deferred_first", [True, False])
def test_weight_shared_with_a_layer_whose_gradient_is_deferred(deferred_first):
    """HipLinear leaves a large weight's gradient as factors for the optimiser's step; the 8-bit product of the same weight adds to
    it, whichever backward runs first."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import model as ym
    from yolo_from_scratch_amd.train import FlatSGD
    torch.manual_seed(12)
    lin = ym.HipLinear(4096, 4096).to(DEV)
    x = torch.randn(2, 70, 4096, device=DEV).bfloat16()
    dy = torch.randn(2, 70, 4096, device=DEV).bfloat16()
    ga, gab = torch.autograd.grad(lin(x[0]), (lin.weight, lin.bias), dy[0])
    gb, gbb = torch.autograd.grad(yfs.fp8_linear(x[1], lin.weight, lin.bias), (lin.weight, lin.bias), dy[1])
    opt = FlatSGD(lin.parameters(), lr=0.1, momentum=0.9)
    lin.weight._yfs_grad_sink.fill_(7)                       # last step's gradient
    opt.zero_grad()
    calls = [lambda: lin(x[0]).backward(dy[0]), lambda: yfs.fp8_linear(x[1], lin.weight, lin.bias).backward(dy[1])]
    for call in calls if deferred_first else calls[::-1]:
        call()
    assert getattr(lin.weight, "_yfs_factors", None) is None
    for got, a, b in ((lin.weight.grad, ga, gb), (lin.bias.grad, gab, gbb)):     # products with sums in fp32, one more rounding
        assert bool(((got - (a + b)).abs() <= 2.0 ** -22 * (a.abs() + b.abs()) + 2.0 ** -24 * 70 * 20).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [129, 4096, 4097, 200704, 1000003])
def test_bias_gradient_over_many_rows(m):
    """The 128-row sums are joined by 32 chains and these in turn, so that what a column loses grows with a 32nd of the rows: 7
    roundings in a tile of 128 rows, one for each 32nd tile, 31 behind them.  Equal values lose most, all in one direction."""
    import yolo_from_scratch_amd as yfs
    c = torch.tensor([1.0, 1.1, 1 / 3, -0.7, 1.0000001, 123.456, -1e-3, 3.3, 0.6, 1.9], device=DEV)
    dy = c.expand(m, 10).contiguous()
    dy[:, 9] = torch.randn(m, device=DEV, generator=torch.Generator(DEV).manual_seed(m))
    x = torch.ones(m, 4, device=DEV)
    w, b = torch.ones(10, 4, device=DEV, requires_grad=True), torch.zeros(10, device=DEV, requires_grad=True)
    _, db = torch.autograd.grad(yfs.fp8_linear(x, w, b), (w, b), dy)
    chain = 7 + -(-(-(-m // 128)) // 32) + 31
    err = (db.double() - dy.double().sum(0)).abs()
    assert bool((err <= chain * 2.0 ** -24 * dy.double().abs().sum(0)).all()), (err / dy.double().abs().sum(0) * 2 ** 24).tolist()
    assert torch.equal(torch.autograd.grad(yfs.fp8_linear(x, w, b), (w, b), dy)[1], db)


def test_tolerance_covers_every_plan():
    """The 96 + K / 32 half steps that the products are held to, from the plans themselves: 32 products in one matrix instruction,
    four instructions for each block of 128 of a part, and one addition for each part (98 of them at 64 x 128 x 50176).  A layer
    that trains with up to 64 rows has at most 128 parts of two blocks or more: 4 K / (128 parts) + parts <= K / 32 there too."""
    import random
    rng = random.Random(8)
    most = 0
    for _ in range(20000):
        m, n, k = [max(1, int(2 ** rng.uniform(0, top))) for top in (15, 17, 17)]
        _, _, parts, per, _ = _plan(m, n, k, torch.float32)
        assert parts == 1 or per >= 4 and parts <= k / 512 + 1, (m, n, k)
        assert 32 + 4 * per + parts - 1 <= 96 + k / 32, (m, n, k)
        most = max(most, parts)
    assert most > 64


@pytest.mark.gpu
def test_second_derivative_in_an_optimisers_arena_is_refused():
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd.train import FlatSGD
    lin = yfs.Fp8Linear(64, 8).to(DEV)
    FlatSGD(lin.parameters(), lr=0.1)
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(lin(x).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_longest_axes(axis):
    """The largest size along each axis, 2^23 - 256: forward, all three gradients, and the served form.  Operands are small whole
    numbers, which 8 bits hold, so that a sum is exact as far as it stays below 2^24.  y of the longest reduction reaches 4 * (2^23 - 256),
    between 2^24 and 2^25: its parts of 256 blocks are below 2^18 and exact, and each of the 256 additions that join them, and the
    bias's, rounds by half a step of 2 at most: 257 half steps, 257 * 2^-24 of the sum at most."""
    import yolo_from_scratch_amd as yfs
    big = (1 << 23) - 256
    m, n, k = [big if i == axis else 1 for i in range(3)]
    i = lambda c, mod: (torch.arange(c, device=DEV) % mod - mod // 2).float()   # noqa: E731
    x = (i(m, 3)[:, None] + i(k, 5)[None]).bfloat16().requires_grad_()
    w = (i(n, 5)[:, None] * (i(k, 3)[None] + 2)).requires_grad_()
    b = i(n, 7).requires_grad_()
    dy = (i(m, 5)[:, None] + i(n, 3)[None]).bfloat16()
    xd, wd, dd = x.detach().double(), w.detach().double(), dy.double()
    y = yfs.fp8_linear(x, w, b)
    ref = xd @ wd.t() + b.detach().double()
    close = lambda got, ref: bool(((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs()).all())   # noqa: E731
    assert close(y.detach(), ref)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert close(dx, dd @ wd) and torch.equal(dw.double(), dd.t() @ xd) and torch.equal(db.double(), dd.sum(0))
    with torch.no_grad():
        wq = yfs.quantize_fp8(w)
        assert torch.equal(wq.dequantize(), w)
        err = (yfs.fp8_matmul(x, wq, b, out_dtype=torch.float32).double() - ref).abs()
        assert bool((err <= (257 * 2.0 ** -24 * ref.abs() if axis == 2 else 0 * ref)).all()) and close(yfs.fp8_matmul(x, wq, b), ref)
