"""The head operators together, as a training step and a server use them: 8-bit linear -> layer norm -> LeakyReLU and dropout
-> 8-bit linear, and the model forms that are built from them."""
import numpy as np
import pytest
import torch

from oracle import head_ref as hr

DEV = "cuda:0"


def _np(t):
    return t.detach().double().cpu().numpy()


def test_model_forms_keep_the_linear_layers_keys():
    from yolo_from_scratch_amd import model as ym
    plain = ym.YoloRegressorModel(head_out=4, image_size=64)
    base = set(plain.state_dict())
    for norm, fp8 in ((True, False), (False, True), (True, True)):
        net = ym.YoloRegressorModel(head_out=4, image_size=64, head_norm=norm, head_fp8=fp8)
        extra = {"fc.2.weight", "fc.2.bias"} if norm else set()
        assert set(net.state_dict()) == base | extra
        net.load_state_dict(plain.state_dict(), strict=not norm)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,out", [(1, 300, 96, 4), (20, 1024, 512, 30), (130, 700, 384, 257)])
def test_chain_forward_and_backward(m, k, n, out):
    """Every stage against the oracle on the values that went into it (one rounding and the fp32 sums of that stage), and the
    chain's gradients equal to those of the stages one after the other, bit for bit."""
    import yolo_from_scratch_amd as yfs
    g = torch.Generator().manual_seed(m)
    rnd = lambda *s: torch.randn(*s, generator=g).to(DEV)   # noqa: E731
    x = rnd(m, k).bfloat16().requires_grad_()
    w1, b1 = (rnd(n, k) / k ** 0.5).requires_grad_(), rnd(n).requires_grad_()
    lw, lb = (1 + 0.1 * rnd(n)).requires_grad_(), (0.1 * rnd(n)).requires_grad_()
    w2, b2 = (rnd(out, n) / n ** 0.5).requires_grad_(), rnd(out).requires_grad_()
    dy = rnd(m, out).bfloat16()
    leaves = (x, w1, b1, lw, lb, w2, b2)

    def chain():
        z = yfs.fp8_linear(x, w1, b1)
        h = yfs.layer_norm(z, lw, lb)
        d = yfs.dropout(h, 0.2, 99, slope=0.1)
        return z, h, d, yfs.fp8_linear(d, w2, b2)
    z, h, d, y = chain()
    whole = torch.autograd.grad(y, leaves, dy)

    u = 2.0 ** -8
    q = lambda t: hr.rounded(_np(t), 1, 128)   # noqa: E731
    qw = lambda t: hr.rounded(_np(t), 128, 128)   # noqa: E731

    def linear_close(got, a, b, bias):
        ref = a @ b.T + bias
        inner = 2.0 ** -9 * np.abs(a).max() * np.abs(b).max() * -(-a.shape[1] // 128) + 1e-5 * (np.abs(a) @ np.abs(b).T + np.abs(bias))
        assert (np.abs(_np(got) - ref) <= u * (np.abs(ref) + inner) + inner).all()
    linear_close(z, q(x), qw(w1), _np(b1))
    ref = hr.layer_norm(_np(z), _np(lw), _np(lb))[0]
    assert (np.abs(_np(h) - ref) <= u * np.abs(ref) + 1e-4).all()
    ref = hr.dropout(_np(h), 0.2, 99, 0.1)
    assert (np.abs(_np(d) - ref) <= u * np.abs(ref)).all() and np.array_equal(_np(d) == 0, ref == 0)
    linear_close(y, q(d), qw(w2), _np(b2))

    d1, h1, z1 = [t.detach().requires_grad_() for t in (d, h, z)]
    gd, gw2, gb2 = torch.autograd.grad(yfs.fp8_linear(d1, w2, b2), (d1, w2, b2), dy)
    gh, = torch.autograd.grad(yfs.dropout(h1, 0.2, 99, slope=0.1), h1, gd)
    gz, glw, glb = torch.autograd.grad(yfs.layer_norm(z1, lw, lb), (z1, lw, lb), gh)
    gx, gw1, gb1 = torch.autograd.grad(yfs.fp8_linear(x, w1, b1), (x, w1, b1), gz)
    for a, b in zip(whole, (gx, gw1, gb1, glw, glb, gw2, gb2)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_training_step_of_the_chain():
    """Forward, backward and a plain update captured together: every replay equals the eager step on the same weights, with a
    new dropout mask each time from a seed in device memory."""
    import yolo_from_scratch_amd as yfs
    torch.manual_seed(3)
    x, t = torch.randn(64, 640, device=DEV).bfloat16(), torch.randn(64, 256, device=DEV)
    seed = torch.tensor([1], device=DEV)

    def fresh():
        gen = torch.Generator().manual_seed(8)
        w = (torch.randn(256, 640, generator=gen) / 25).to(DEV).requires_grad_()
        return w, torch.ones(256, device=DEV, requires_grad=True)

    def step(w, lw):
        y = yfs.dropout(yfs.layer_norm(yfs.fp8_linear(x, w), lw), 0.1, seed, slope=0.1)
        loss = (y.float() - t).square().mean()
        gw, gl = torch.autograd.grad(loss, (w, lw))
        with torch.no_grad():
            w.sub_(gw, alpha=0.5)
            lw.sub_(gl, alpha=0.5)
        return loss.detach()
    we, le = fresh()
    eager = []
    for k in range(5):
        seed.fill_(100 + k)
        eager.append(float(step(we, le)))
    wc, lc = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*fresh())                                     # warm-up, on other leaves
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = step(wc, lc)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(5):
        seed.fill_(100 + k)
        graph.replay()
        torch.cuda.synchronize()
        assert float(loss) == eager[k], k
    assert torch.equal(wc, we) and torch.equal(lc, le)


@pytest.mark.gpu
@pytest.mark.parametrize("norm,fp8", [(True, False), (False, True), (True, True)])
def test_model_forms_train_and_serve(norm, fp8):
    """The model with the new head through train_one_epoch with FlatSGD, evaluate, a frozen copy for serving."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import model as ym
    from yolo_from_scratch_amd.train import FlatSGD, evaluate, train_one_epoch
    torch.manual_seed(0)
    net = ym.YoloRegressorModel(head_out=4, image_size=64, head_norm=norm, head_fp8=fp8).to(DEV)
    opt = FlatSGD(net.parameters(), lr=1e-3, momentum=0.9)
    before = {k: v.detach().clone() for k, v in net.named_parameters()}
    data = [(torch.rand(6, 3, 64, 64), torch.rand(6, 4)) for _ in range(3)]
    assert np.isfinite(train_one_epoch(net, data, DEV, opt, None, yfs.MSELoss(), max_norm=1.0))
    for k, p in net.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[k]), k
    loss, iou = evaluate(net, data, DEV, yfs.MSELoss())
    assert np.isfinite(loss) and 0 <= iou <= 1
    with torch.no_grad():
        x = data[0][0].to(DEV)
        want = net(x)
        state = {k: v.clone() for k, v in net.state_dict().items()}
        served = yfs.freeze_fp8(net)
        got = served(x)
        assert got.shape == want.shape and torch.equal(served(x), got)
        if fp8:      # the same 8-bit products; fc.1's few rows are summed by another kernel: one rounding of bf16 and its 8-bit echo
            assert float((got - want).abs().max()) <= 2.0 ** -3 * float(want.abs().max()) + 1e-2
        assert torch.isfinite(got).all()
        one = served(x[:1])                                 # a single image, and a batch of the same one
        assert torch.isfinite(one).all()
    assert "fc.1.weight" in state and "fc.1.weight_data" in dict(served.named_buffers())


@pytest.mark.gpu
def test_feature_map_norm_behind_a_conv_block():
    """HipLayerNorm(channels_first) takes a conv block's channels-last map as it is and keeps its layout, forward and backward."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import model as ym
    torch.manual_seed(1)
    block, norm = ym.Conv2D(64, 128, 3).to(DEV), yfs.HipLayerNorm(128, channels_first=True).to(DEV)
    x = torch.randn(2, 64, 14, 14, device=DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
    f = block(x)
    y = norm(f)
    assert y.is_contiguous(memory_format=torch.channels_last)
    ref = hr.layer_norm(_np(f.permute(0, 2, 3, 1)).reshape(-1, 128))[0]
    assert (np.abs(_np(y.permute(0, 2, 3, 1)).reshape(-1, 128) - ref) <= 2.0 ** -8 * np.abs(ref) + 1e-4).all()
    y.float().square().sum().backward()
    for p in [x, *block.parameters(), *norm.parameters()]:
        assert p.grad is not None and torch.isfinite(p.grad).all()


def test_forward_mode_derivatives_are_refused():
    """A tangent of forward-mode differentiation is refused, not dropped, whichever argument carries it and whether or not the
    tensor requires a gradient."""
    import torch.autograd.forward_ad as fwd
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd.fp8_ops import _pad
    n, k = 40, 200
    data = torch.zeros(n, _pad(k), dtype=torch.uint8).view(torch.float8_e4m3fn)
    w8 = yfs.Fp8Tensor(data, torch.full((1, 2), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu), k)
    lin = yfs.Fp8Linear(k, n)
    lin.weight._yfs_grad_sink = torch.zeros(n, k)
    x, w, wk, b = torch.zeros(3, k), torch.zeros(n, k), torch.ones(k), torch.zeros(n)
    with fwd.dual_level():
        for grad in (False, True):
            dual = lambda t: fwd.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))   # noqa: E731
            for call in (lambda: yfs.layer_norm(dual(x)), lambda: yfs.layer_norm(x, dual(wk)), lambda: yfs.layer_norm(x, wk, dual(wk)),
                         lambda: yfs.dropout(dual(x), 0.5, 1), lambda: yfs.fp8_linear(dual(x), w), lambda: yfs.fp8_linear(x, dual(w)),
                         lambda: yfs.fp8_linear(x, w, dual(b)), lambda: yfs.fp8_linear(dual(x), lin.weight, lin.bias),
                         lambda: yfs.fp8_matmul(dual(x), w8), lambda: yfs.fp8_matmul(x, w8, dual(b)), lambda: yfs.quantize_fp8(dual(w))):
                with pytest.raises(yfs.YfsError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(yfs.YfsError, match="forward-mode"):
                    call()
        for call in (lambda: yfs.layer_norm(x), lambda: yfs.dropout(x, 0.5, 1), lambda: yfs.fp8_linear(x, w), lambda: yfs.fp8_matmul(x, w8)):
            with pytest.raises(yfs.YfsError, match="CPU tensor"):      # (no tangent: the next refusal)
                call()


@pytest.mark.gpu
def test_create_graph_is_refused_by_the_backward_pass_itself():
    import yolo_from_scratch_amd as yfs
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    w = torch.ones(8, 32, device=DEV, requires_grad=True)
    for f in (lambda: yfs.layer_norm(x), lambda: yfs.dropout(x, 0.5, 1), lambda: yfs.fp8_linear(x, w)):
        y = f().sum()
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y, x, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_frozen_form_of_a_head_trained_in_16_bits(norm):
    """Every stage of the frozen head is the 8-bit product of its quantised weight, with its bias and its activation, and fc.1 stays
    within the two roundings to e4m3 of its 16-bit form: half a step of 2^-3 each and their product, 2^-10 of the largest value
    of a block (x: of the row's, w: of the 128 x 128 block's) for what lies in the subnormal range, then the 16-bit sums' own error."""
    import yolo_from_scratch_amd as yfs
    from yolo_from_scratch_amd import model as ym
    torch.manual_seed(4)
    net = ym.YoloRegressorModel(head_out=30, image_size=64, head_norm=norm).to(DEV).eval()
    with torch.no_grad():
        for i in (1, 4):
            net.fc[i].bias.normal_()
        if norm:
            net.fc[2].weight.uniform_(0.5, 1.5), net.fc[2].bias.normal_()
        x = torch.rand(6, 3, 64, 64, device=DEV)
        flat = net.feat(x).flatten(1)
        w1, b1, w4, b4 = [t.detach().clone() for i in (1, 4) for t in (net.fc[i].weight, net.fc[i].bias)]
        plain, hidden16 = net(x), net.fc[1](flat).float()
        q1, q4 = yfs.quantize_fp8(w1), yfs.quantize_fp8(w4)
        served = yfs.freeze_fp8(net)
        assert torch.equal(served.feat(x).flatten(1), flat)
        slope = None if norm else ym.SLOPE
        h = yfs.fp8_matmul(flat, q1, b1, slope, torch.bfloat16)
        assert torch.equal(served.fc[1](flat), h)
        if norm:
            a = yfs.dropout(yfs.layer_norm(h, net.fc[2].weight, net.fc[2].bias), 0.0, 0, ym.SLOPE)
        else:
            a = h
        want = yfs.fp8_matmul(a, q4, b4, None, torch.bfloat16).float()
        assert torch.equal(served(x), want) and not torch.equal(want, plain)

    f, w = _np(flat), _np(w1)
    k = f.shape[1]
    top = lambda t: np.abs(t).reshape(t.shape[0], k // 128, 128).max(2)   # noqa: E731
    fe = np.abs(f) * 2.0 ** -4 + np.repeat(top(f), 128, 1) * 2.0 ** -17      # half a subnormal step is 2^-10 s, and s < max / 224
    wt = top(w).reshape(-1, 128, k // 128).max(1)                           # of a 128 x 128 block
    we = np.abs(w) * 2.0 ** -4 + np.repeat(np.repeat(wt, 128, 0), 128, 1) * 2.0 ** -17
    bound = np.abs(f) @ we.T + fe @ np.abs(w).T + fe @ we.T
    bound += np.abs(f) @ np.abs(w).T * 2.0 ** -8 + 2.0 ** -7 * np.abs(_np(hidden16))     # bf16 weights and results, the 8-bit sums
    ref = f @ w.T + _np(b1)
    if slope is not None:
        ref = np.where(ref > 0, ref, slope * ref)
    for got in (_np(h), _np(hidden16)):
        assert (np.abs(got - ref) <= bound + 2.0 ** -7 * np.abs(ref) + 1e-6).all()
